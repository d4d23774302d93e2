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

#include <atomic>

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
// Row kernel: the state streams through registers once, T tokens applied in
// order. For single tokens it moves 8 N bytes of state per channel against
// some 8 bytes of activations, so HBM bounds it. Four states (16 bytes) a
// thread: a warp's accesses are contiguous, and y takes a butterfly over the
// N/4 lanes of a channel.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 128;

// A as a power of two's exponent; finite, so that a step of zero keeps the
// state even where A is -inf.
__device__ __forceinline__ float scaled(float a) { return fmaxf(a * kLog2e, -FLT_MAX); }

template <typename T, int N>
__global__ void __launch_bounds__(kRowThreads) scan_rows_kernel(ScanArgs p) {
  constexpr int LPC = N / 4;  // lanes of a channel
  constexpr int CPB = kRowThreads / LPC;
  const int cblocks = (p.D + CPB - 1) / CPB;
  const int n = blockIdx.x / cblocks;
  const int lane = threadIdx.x % LPC;
  const int d = (blockIdx.x - n * cblocks) * CPB + threadIdx.x / LPC;
  int64_t row;
  const SeqSpan sp = seq_span(p.seqs, n);
  if (!state_row(p.ids, p.num_slots, n, &row)) {
    if (threadIdx.x == 0) report(p.status, WKVM_ERR_SLOT_RANGE);
    return;
  }
  if (!sp.ok) {
    if (threadIdx.x == 0) report(p.status, WKVM_ERR_INVALID_ARG);
    return;
  }
  const bool on = d < p.D;  // the butterfly needs every lane
  const int dc = on ? d : p.D - 1;
  const int64_t hoff = (row * p.D + dc) * N + lane * 4;
  float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.h_in) h = ld_stream_f4(p.h_in + hoff);
  float4 a = *reinterpret_cast<const float4*>(p.A + (int64_t)dc * N + lane * 4);
  a.x = scaled(a.x); a.y = scaled(a.y); a.z = scaled(a.z); a.w = scaled(a.w);
  const float bias = p.bias ? p.bias[dc] : 0.f, skip = p.skip ? p.skip[dc] : 0.f;
  const int g = dc / (p.D / p.G);
  const T* xp = static_cast<const T*>(p.x.p) + act_row(p.seqs, p.x, n, sp.bos) + dc;
  const T* dp = static_cast<const T*>(p.dt.p) + act_row(p.seqs, p.dt, n, sp.bos) + dc;
  const T* bp = static_cast<const T*>(p.B.p) + act_row(p.seqs, p.B, n, sp.bos) + g * N + lane * 4;
  const T* cp = static_cast<const T*>(p.C.p) + act_row(p.seqs, p.C, n, sp.bos) + g * N + lane * 4;
  const T* zp = p.z.p ? static_cast<const T*>(p.z.p) + act_row(p.seqs, p.z, n, sp.bos) + dc : nullptr;
  T* op = static_cast<T*>(p.o) + sp.bos * p.D + dc;
  for (int64_t t = 0; t < sp.len; ++t) {
    const float x = to_f32(xp[t * p.x.ts]);
    float delta = to_f32(dp[t * p.dt.ts]) + bias;
    if (p.softplus) delta = softplus(delta);
    float bv[4], cv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bv[i] = to_f32(bp[t * p.B.ts + i]);
      cv[i] = to_f32(cp[t * p.C.ts + i]);
    }
    const float z = zp ? to_f32(zp[t * p.z.ts]) : 0.f;
    const float dx = delta * x;
    h.x = fmaf(ex2(delta * a.x), h.x, dx * bv[0]);
    h.y = fmaf(ex2(delta * a.y), h.y, dx * bv[1]);
    h.z = fmaf(ex2(delta * a.z), h.z, dx * bv[2]);
    h.w = fmaf(ex2(delta * a.w), h.w, dx * bv[3]);
    float y = fmaf(h.x, cv[0], h.y * cv[1]) + fmaf(h.z, cv[2], h.w * cv[3]);
#pragma unroll
    for (int off = LPC / 2; off > 0; off >>= 1) y += __shfl_xor_sync(0xffffffffu, y, off);
    y = fmaf(skip, x, y);
    if (zp) y *= silu<true>(z);
    if (on && lane == 0) op[t * p.D] = from_f32<T>(y);
  }
  if (on && p.h_out) st_stream_f4(p.h_out + hoff, h);
}

// ---------------------------------------------------------------------------
// Tile kernel, for prompts. T D N exponentials (16 a clock and SM) bound it:
// 16 states give 4.65e12 / s against 8 bytes of activations per 16 of them.
//
// One CTA walks one sequence for CB channels, kTT tokens at a time. Each
// thread keeps NS states of one channel; the L = N / NS threads of a channel
// leave their partial sums of C h in shared memory and the thread that owns
// the output element adds them. What is per (token, channel) - softplus, the
// skip, the gate, conversions - is done once by the owner of the element, not
// by the L threads: they read (delta, delta x) pairs. Inputs of the next tile
// are in registers while this one runs.
//
// Few rows (a long prompt alone, few channels): the CTAs of a cluster split
// the sequence's tiles between them. Each first runs its part from a zero
// state for its final state and the sum of its steps (whose exponential is
// the part's whole decay, A being constant), then takes the parts before it
// from its peers' shared memory and runs its part again from its true start.
// ---------------------------------------------------------------------------
constexpr int kTT = 32;

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

template <typename T, int V> struct alignas(sizeof(T) * V) Raw { T e[V]; };

// V elements at p, of which the first `n` exist (the others read as zero).
// vec: p is aligned to the whole vector and n is 0 or at least V.
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p, int n, bool vec) {
  Raw<T, V> r;
  if (vec && n >= V) return *reinterpret_cast<const Raw<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) r.e[i] = i < n ? p[i] : from_f32<T>(0.f);
  return r;
}

constexpr int min_i(int a, int b) { return a < b ? a : b; }

template <int N, int NS, int NT>
struct Tile {
  static constexpr int L = N / NS;                  // threads of a channel
  static constexpr int CB = NT / L;                 // channels of a CTA
  static constexpr int TP = 4 / NS;                 // tokens in one 16-byte read of B or C
  static constexpr int EPT = kTT * CB / NT;         // elements of x a thread owns
  static constexpr int VE = min_i(EPT, 4), RV = EPT / VE;
  static constexpr int BPT = kTT * N / NT;          // elements of B a thread loads
  static constexpr int VB = min_i(BPT, 4), RB = BPT / VB;
  static constexpr int YROW = NT + NT / 8;          // 4 floats of padding every 32: no bank conflicts
  // shared memory, in floats
  static constexpr int oD = 0;                      // [kTT / TP][CB][TP] (delta, delta x)
  static constexpr int oB = oD + 2 * kTT * CB;      // [kTT / TP][L][TP][NS]
  static constexpr int oC = oB + kTT * N;
  static constexpr int oY = oC + kTT * N;           // [kTT][YROW] partial sums
  static constexpr int oH = oY + kTT * YROW;        // cluster: final states [NS][NT], step sums [NT]
  static constexpr int bytes(bool cluster) { return 4 * (oH + (cluster ? (NS + 1) * NT : 0)); }
  static_assert(EPT >= 1 && BPT >= 1 && CB >= 1, "tile too small for the block");
};

struct TileArgs {
  ScanArgs s;
  int32_t cblocks;   // channel blocks of a group
  int32_t parts;     // CTAs of a cluster (1: none)
  bool vec_x, vec_b; // whole-vector accesses to x, dt, z, o and to B, C
  bool longest_first;
};

template <typename T, int N, int NS, int NT, bool CLUSTER>
__global__ void __launch_bounds__(NT) scan_tiles_kernel(TileArgs q) {
  using K = Tile<N, NS, NT>;
  constexpr int L = K::L, CB = K::CB, TP = K::TP, VE = K::VE, RV = K::RV, VB = K::VB, RB = K::RB;
  constexpr int CBV = CB / VE;
  extern __shared__ __align__(16) float sm[];
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
    __syncthreads();
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

  // ---- this thread's states and its channel's A
  const bool on = ch < cn;
  const int64_t hoff = (row * p.D + c0 + (on ? ch : 0)) * N + lane * NS;
  f32x2 h[NS / 2], a[NS / 2];
  float hs[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) hs[i] = p.h_in ? p.h_in[hoff + i] : 0.f;
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) {
    const float* ap = p.A + (int64_t)(c0 + (on ? ch : 0)) * N + lane * NS + 2 * i;
    a[i] = pack2(scaled(ap[0]), scaled(ap[1]));
    h[i] = pack2(hs[2 * i], hs[2 * i + 1]);
  }

  // ---- the elements of a tile this thread owns: channels ce..ce+VE-1 of
  //      tokens te + r * TS
  const int te = tid / CBV, ce = (tid % CBV) * VE;
  constexpr int TS = NT / CBV;
  const int nv = cn - ce;  // channels of the vector that exist
  float bias[VE], skip[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    bias[i] = p.bias && i < nv ? p.bias[c0 + ce + i] : 0.f;
    skip[i] = p.skip && i < nv ? p.skip[c0 + ce + i] : 0.f;
  }
  const T* xp = static_cast<const T*>(p.x.p) + act_row(p.seqs, p.x, n, sp.bos) + c0 + ce;
  const T* dp = static_cast<const T*>(p.dt.p) + act_row(p.seqs, p.dt, n, sp.bos) + c0 + ce;
  const T* zp = p.z.p ? static_cast<const T*>(p.z.p) + act_row(p.seqs, p.z, n, sp.bos) + c0 + ce : nullptr;
  const T* bp = static_cast<const T*>(p.B.p) + act_row(p.seqs, p.B, n, sp.bos) + g * N;
  const T* cp = static_cast<const T*>(p.C.p) + act_row(p.seqs, p.C, n, sp.bos) + g * N;
  T* op = static_cast<T*>(p.o) + sp.bos * p.D + c0 + ce;

  Raw<T, VE> rx[RV], rd[RV], rz[RV];
  Raw<T, VB> rb[RB], rc[RB];
  auto fetch = [&](int64_t t0, bool emit) {
#pragma unroll
    for (int r = 0; r < RV; ++r) {
      const int64_t t = t0 + te + r * TS;
      const int k = t < sp.len ? nv : 0;
      rx[r] = load_raw<T, VE>(xp + t * p.x.ts, k, q.vec_x);
      rd[r] = load_raw<T, VE>(dp + t * p.dt.ts, k, q.vec_x);
      if (emit && zp) rz[r] = load_raw<T, VE>(zp + t * p.z.ts, k, q.vec_x);
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int e = (r * NT + tid) * VB;
      const int64_t t = t0 + e / N;
      const int k = t < sp.len ? VB : 0;
      rb[r] = load_raw<T, VB>(bp + t * p.B.ts + e % N, k, q.vec_b);
      if (emit) rc[r] = load_raw<T, VB>(cp + t * p.C.ts + e % N, k, q.vec_b);
    }
  };

  float steps = 0.f;  // sum of delta over the part (first pass of a cluster)
  auto run = [&](int64_t t0, int64_t t1, bool emit) {
    if (t0 >= t1) return;
    fetch(t0, emit);
    for (; t0 < t1; t0 += kTT) {
      Raw<T, VE> cx[RV], cz[RV];
#pragma unroll
      for (int r = 0; r < RV; ++r) {
        cx[r] = rx[r];
        cz[r] = rz[r];
        const int t = te + r * TS;
        const bool live = t0 + t < sp.len;
        float* dst = sm + K::oD + 2 * ((t / TP) * CB * TP + (t % TP));
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          float d = to_f32(rd[r].e[i]) + bias[i];
          if (p.softplus) d = softplus(d);
          if (!live) d = 0.f;  // decay 1, input 0
          *reinterpret_cast<float2*>(dst + 2 * TP * (ce + i)) = make_float2(d, live ? d * to_f32(cx[r].e[i]) : 0.f);
        }
      }
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const int e = (r * NT + tid) * VB;
#pragma unroll
        for (int i = 0; i < VB; ++i) {
          const int t = (e + i) / N, s = (e + i) % N;
          const int at = (((t / TP) * L + s / NS) * TP + t % TP) * NS + s % NS;
          sm[K::oB + at] = to_f32(rb[r].e[i]);
          if (emit) sm[K::oC + at] = to_f32(rc[r].e[i]);
        }
      }
      __syncthreads();
      if (t0 + kTT < t1) fetch(t0 + kTT, emit);
      const int live = (int)(sp.len - t0 < kTT ? sp.len - t0 : kTT);
      const float* sD = sm + K::oD + 2 * TP * ch;
      const float* sB = sm + K::oB + 4 * lane;
      const float* sC = sm + K::oC + 4 * lane;
      float* sY = sm + K::oY + tid + (tid >> 5) * 4;
      for (int tb = 0; tb < live; tb += 8) {
#pragma unroll
        for (int u = 0; u < 8; u += TP) {
          const int t = tb + u;
          float dd[2 * TP];
          if constexpr (TP == 2)
            *reinterpret_cast<float4*>(dd) = *reinterpret_cast<const float4*>(sD + 2 * CB * t);
          else
            *reinterpret_cast<float2*>(dd) = *reinterpret_cast<const float2*>(sD + 2 * CB * t);
          const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(sB + (t / TP) * 4 * L);
          ulonglong2 cc = make_ulonglong2(0, 0);
          if (emit) cc = *reinterpret_cast<const ulonglong2*>(sC + (t / TP) * 4 * L);
#pragma unroll
          for (int v = 0; v < TP; ++v) {
            const f32x2 d2 = pack2(dd[2 * v], dd[2 * v]), x2 = pack2(dd[2 * v + 1], dd[2 * v + 1]);
            f32x2 y2 = 0;
#pragma unroll
            for (int i = 0; i < NS / 2; ++i) {
              const f32x2 b2 = (v * (NS / 2) + i) ? bb.y : bb.x, c2 = (v * (NS / 2) + i) ? cc.y : cc.x;
              const float2 e = unpack2(mul2(a[i], d2));
              h[i] = fma2(pack2(ex2(e.x), ex2(e.y)), h[i], mul2(x2, b2));
              y2 = i ? fma2(h[i], c2, y2) : mul2(h[i], c2);
            }
            if (emit) {
              const float2 y = unpack2(y2);
              sY[(t + v) * K::YROW] = y.x + y.y;
            } else {
              steps += dd[2 * v];
            }
          }
        }
      }
      __syncthreads();
      if (!emit) continue;
#pragma unroll
      for (int r = 0; r < RV; ++r) {
        const int t = te + r * TS;
        if (t0 + t >= sp.len) continue;
        const float* src = sm + K::oY + t * K::YROW + ce * L + ((ce * L) >> 5) * 4;
        Raw<T, VE> out;
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          float y = 0.f;
#pragma unroll
          for (int j = 0; j < L; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(src + (i * L + j) + ((i * L + j) >> 5) * 4);
            y += (f.x + f.y) + (f.z + f.w);
          }
          y = fmaf(skip[i], to_f32(cx[r].e[i]), y);
          if (zp) y *= silu<sizeof(T) == 4>(to_f32(cz[r].e[i]));
          out.e[i] = from_f32<T>(y);
        }
        T* dst = op + (t0 + t) * p.D;
        if (q.vec_x && nv >= VE) {
          *reinterpret_cast<Raw<T, VE>*>(dst) = out;
        } else {
#pragma unroll
          for (int i = 0; i < VE; ++i)
            if (i < nv) dst[i] = out.e[i];
        }
      }
    }
  };

  if constexpr (CLUSTER) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int64_t tiles = (sp.len + kTT - 1) / kTT, each = (tiles + q.parts - 1) / q.parts * kTT;
    const int64_t b0 = part * each < sp.len ? part * each : sp.len;
    const int64_t b1 = b0 + each < sp.len ? b0 + each : sp.len;
    f32x2 start[NS / 2];
#pragma unroll
    for (int i = 0; i < NS / 2; ++i) {
      start[i] = h[i];
      h[i] = 0;
    }
    if (part + 1 < q.parts) run(b0, b1, false);  // nobody follows the last part
    float* sH = sm + K::oH;
#pragma unroll
    for (int i = 0; i < NS / 2; ++i) {
      const float2 v = unpack2(h[i]);
      sH[(2 * i) * NT + tid] = v.x;
      sH[(2 * i + 1) * NT + tid] = v.y;
    }
    sH[NS * NT + tid] = steps;
    cluster.sync();
    for (int j = 0; j < part; ++j) {
      const float* peer = cluster.map_shared_rank(sH, j);
      const float sum = peer[NS * NT + tid];
#pragma unroll
      for (int i = 0; i < NS / 2; ++i) {
        const float2 e = unpack2(mul2(a[i], pack2(sum, sum)));
        start[i] = fma2(pack2(ex2(e.x), ex2(e.y)), start[i], pack2(peer[(2 * i) * NT + tid], peer[(2 * i + 1) * NT + tid]));
      }
    }
    cluster.sync();  // peers have read; the state row may be written now
#pragma unroll
    for (int i = 0; i < NS / 2; ++i) h[i] = start[i];
    run(b0, b1, true);
    if (part + 1 < q.parts) return;
  } else {
    run(0, sp.len, true);
  }
  if (on && p.h_out) {
#pragma unroll
    for (int i = 0; i < NS / 2; ++i) {
      const float2 v = unpack2(h[i]);
      p.h_out[hoff + 2 * i] = v.x;
      p.h_out[hoff + 2 * i + 1] = v.y;
    }
  }
}

template <typename T, int N>
int launch_rows(const ScanArgs& a, cudaStream_t st) {
  constexpr int CPB = kRowThreads / (N / 4);
  const int64_t blocks = (int64_t)a.seqs.nseq * ((a.D + CPB - 1) / CPB);
  if (blocks > INT32_MAX) return WKVM_ERR_SHAPE;
  scan_rows_kernel<T, N><<<(unsigned)blocks, kRowThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

// Allows a kernel its shared memory (and clusters of 16) on the current
// device, once each.
template <auto Kernel>
int allow(int bytes, bool big_cluster) {
  static std::atomic<uint64_t> done{0};  // a bit per device
  int dev = 0;
  WKVM_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1)) return WKVM_OK;
  WKVM_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (big_cluster)
    WKVM_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return WKVM_OK;
}

template <typename T, int N>
int launch_tiles(const ScanArgs& s, cudaStream_t st) {
  // two states a thread keep two warps on every scheduler at a few thousand
  // channels of one sequence; 128 states would need two warps per channel
  constexpr int NS = N == 128 ? 4 : 2, NT = 256;
  using K = Tile<N, NS, NT>;
  TileArgs q{s, 0, 1, false, false, false};
  const int per_group = s.D / s.G;
  q.cblocks = (per_group + K::CB - 1) / K::CB;
  const int64_t jobs = (int64_t)s.seqs.nseq * q.cblocks * s.G;
  constexpr uintptr_t ax = sizeof(T) * K::VE, ab = sizeof(T) * K::VB;
  auto even = [](const Act& a, int v) { return a.bs % v == 0 && a.ts % v == 0; };
  q.vec_x = per_group % K::VE == 0 && even(s.x, K::VE) && even(s.dt, K::VE) && aligned_to(s.x.p, ax) &&
            aligned_to(s.dt.p, ax) && aligned_to(s.o, ax) &&
            (!s.z.p || (even(s.z, K::VE) && aligned_to(s.z.p, ax)));
  q.vec_b = even(s.B, K::VB) && even(s.C, K::VB) && aligned_to(s.B.p, ab) && aligned_to(s.C.p, ab);
  q.longest_first = s.seqs.cu && s.seqs.nseq > 1 && s.seqs.nseq <= 256;
  // split sequences in time when the whole ones would leave most SMs idle:
  // a split pays twice for the exponentials, so two parts gain nothing
  const int64_t tokens = s.seqs.cu ? s.seqs.T / s.seqs.nseq : s.seqs.T;
  int parts = 1;
  while (parts < 16 && jobs * parts * 2 <= 296 && tokens >= (int64_t)parts * 2 * 2 * kTT) parts *= 2;
  if (parts < 4) parts = 1;
  if (jobs * parts > INT32_MAX) return WKVM_ERR_SHAPE;
  q.parts = parts;
  if (parts == 1) {
    constexpr auto kern = scan_tiles_kernel<T, N, NS, NT, false>;
    if (int rc = allow<kern>(K::bytes(false), false)) return rc;
    kern<<<(unsigned)jobs, NT, K::bytes(false), st>>>(q);
    return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
  }
  constexpr auto kern = scan_tiles_kernel<T, N, NS, NT, true>;
  if (int rc = allow<kern>(K::bytes(true), true)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(jobs * parts));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = K::bytes(true);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, q) == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

template <typename T, int N>
int launch_scan_n(const ScanArgs& a, cudaStream_t st) {
  // a few tokens of every row: the state's traffic decides, so the row kernel
  if (!a.seqs.cu && a.seqs.T <= 8) return launch_rows<T, N>(a, st);
  return launch_tiles<T, N>(a, st);
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
