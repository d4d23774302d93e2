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
  a.x *= kLog2e; a.y *= kLog2e; a.z *= kLog2e; a.w *= kLog2e;
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

template <typename T, int N>
int launch_scan_n(const ScanArgs& a, cudaStream_t st) {
  constexpr int CPB = kRowThreads / (N / 4);
  const int64_t blocks = (int64_t)a.seqs.nseq * ((a.D + CPB - 1) / CPB);
  if (blocks > INT32_MAX) return WKVM_ERR_SHAPE;
  scan_rows_kernel<T, N><<<(unsigned)blocks, kRowThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
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

ScanArgs scan_args(const void* x, const void* dt, const float* A, const void* B, const void* C,
                   const float* skip, const void* z, const float* dt_bias, void* o,
                   const int64_t* s, const int64_t* cu, int32_t nseq, int32_t T, int32_t D,
                   int32_t G, int32_t softplus, int32_t* status) {
  return {{x, s[0], s[1]}, {dt, s[2], s[3]}, {z, s[4], s[5]}, {B, s[6], s[7]}, {C, s[8], s[9]},
          A, skip, dt_bias, o, nullptr, nullptr, nullptr, 0, {cu, nseq, T}, D, G, softplus, status};
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
