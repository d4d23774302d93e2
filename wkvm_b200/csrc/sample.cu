// Choice of one token per row of logits from a given uniform number, under
// temperature, top-k, top-p and min-p. For row b with maximum m:
//
//   w_i = exp((l_i - m) / T)                              (T = 0: greedy)
//   top-k keeps the k largest l_i (ties: the lowest ids)
//   top-p keeps, of those in descending order (ties: the lowest ids first),
//     the shortest prefix whose mass is >= p times the mass of those
//   min-p keeps, of those, w_i >= min_p (the largest w is 1)
//   token = first kept id whose running mass, in order of ids, is > u Z, with
//     Z the mass kept; logprob = log(w_token / Z)
//
// -inf and NaN logits are never kept; logits of +inf share the whole mass. A
// row with nothing to keep gives token -1 and logprob -inf.
//
// Masses are fp64: where one token ends and the next begins moves by the
// error of a running mass, and with 65,536 tokens an error of 1e-7 would
// change about one row's token in two hundred.
#include "common.cuh"

namespace wkvm {
namespace {

struct SampleArgs {
  const void* logits;
  int64_t row_stride;  // elements
  const float* u;
  const float *temperature, *top_p, *min_p;  // per row, or null: the value below
  const int32_t* top_k;
  float temperature0, top_p0, min_p0;
  int32_t top_k0;
  int64_t* token;
  float* logprob;
  int32_t B, V;
  int* status;
};

// Ascending unsigned order of floats; NaN and -inf become 0 (never kept).
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 sorts as +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

constexpr int kThreads = 1024;

template <typename V, typename F>
__device__ V block_sum(V x, V* scratch, F) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  V s = 0;
  for (int i = 0; i < kThreads / 32; ++i) s += scratch[i];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs p) {
  __shared__ double sd[kThreads / 32];
  __shared__ int si[kThreads / 32];
  __shared__ int s_token;
  const int b = blockIdx.x, tid = threadIdx.x, V = p.V;
  const T* row = static_cast<const T*>(p.logits) + b * p.row_stride;
  float temp = p.temperature ? p.temperature[b] : p.temperature0;
  int k = p.top_k ? p.top_k[b] : p.top_k0;
  const double tp = p.top_p ? p.top_p[b] : p.top_p0, mp = p.min_p ? p.min_p[b] : p.min_p0;
  const double u = p.u[b];
  if (!(temp > 0.f)) { temp = 1.f; k = 1; }
  const double inv_t = 1.0 / (double)temp;
  auto key = [&](int i) { return key_of(to_f32(row[i])); };
  auto isum = [&](int x) { return block_sum<int>(x, si, 0); };
  auto dsum = [&](double x) { return block_sum<double>(x, sd, 0); };

  // the largest key and how many logits can be kept at all
  uint32_t mk = 0;
  int n = 0;
  for (int i = tid; i < V; i += kThreads) {
    const uint32_t q = key(i);
    mk = max(mk, q);
    n += q != 0;
  }
  n = isum(n);
  __shared__ unsigned s_mk;
  if (tid == 0) { s_mk = 0; s_token = -1; }
  __syncthreads();
  atomicMax(&s_mk, mk);
  __syncthreads();
  mk = s_mk;
  if (n == 0) {
    if (tid == 0) { p.token[b] = -1; p.logprob[b] = -INFINITY; }
    return;
  }
  const double m = value_of(mk);
  auto weight = [&](uint32_t q) -> double {
    if (q == 0) return 0.0;
    if (q == mk) return 1.0;
    if (isinf(m)) return 0.0;
    return exp(((double)value_of(q) - m) * inv_t);
  };

  // kept: key > tau, or key == tau and id < lim (always a prefix of the
  // descending order)
  uint32_t tau = 0;
  int lim = 0;  // key 0 is never kept
  auto kept = [&](uint32_t q, int i) { return q > tau || (q == tau && i < lim); };
  auto limit_ids = [&](uint32_t key_eq, int budget) {  // id bound that keeps `budget` ties
    int lo = 0, hi = V;
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      int c = 0;
      for (int i = tid; i < mid; i += kThreads) c += key(i) == key_eq;
      c = isum(c);
      if (c >= budget) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  if (k > 0 && k < n) {
    uint32_t lo = 1, hi = mk;  // largest key with at least k keys >= it
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      int c = 0;
      for (int i = tid; i < V; i += kThreads) c += key(i) >= mid;
      c = isum(c);
      if (c >= k) lo = mid; else hi = mid - 1;
    }
    int above = 0;
    for (int i = tid; i < V; i += kThreads) above += key(i) > lo;
    above = isum(above);
    lim = limit_ids(lo, k - above);
    tau = lo;
  }
  auto mass_from = [&](uint32_t from) {  // mass of what is kept with key >= from
    double s = 0;
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t q = key(i);
      if (q >= from && kept(q, i)) s += weight(q);
    }
    return dsum(s);
  };
  if (tp < 1.0) {
    const double goal = tp * mass_from(0);
    uint32_t lo = 1, hi = mk;
    while (lo < hi) {  // largest key with mass >= goal at or above it
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if (mass_from(mid) >= goal) lo = mid; else hi = mid - 1;
    }
    const double above = lo == 0xffffffffu ? 0.0 : mass_from(lo + 1);
    int ties = 0;
    for (int i = tid; i < V; i += kThreads) {
      const uint32_t q = key(i);
      ties += q == lo && kept(q, i);
    }
    ties = isum(ties);
    const double w = weight(lo);
    int take = 1;
    while (take < ties && above + take * w < goal) ++take;
    lim = limit_ids(lo, take);
    tau = lo;
  }
  // draw: contiguous ids per thread
  const int per = (V + kThreads - 1) / kThreads;
  const int i0 = min(V, tid * per), i1 = min(V, i0 + per);
  auto share = [&](int i) {
    const uint32_t q = key(i);
    if (!kept(q, i)) return 0.0;
    const double w = weight(q);
    return w >= mp || q == mk ? w : 0.0;
  };
  double mine = 0;
  for (int i = i0; i < i1; ++i) mine += share(i);
  __shared__ double s_mass[kThreads];
  s_mass[tid] = mine;
  __syncthreads();
  if (tid == 0) {
    double z = 0;
    for (int t = 0; t < kThreads; ++t) z += s_mass[t];
    const double goal = u * z;
    double c = 0, wt = 0;
    int tok = -1;
    for (int t = 0; t < kThreads && (tok < 0 || c <= goal); ++t) {
      if (s_mass[t] == 0.0) continue;
      if (c + s_mass[t] <= goal && t * per + per < V) {
        bool later = false;
        for (int r = t + 1; r < kThreads; ++r) later |= s_mass[r] > 0.0;
        if (later) { c += s_mass[t]; continue; }
      }
      const int a0 = min(V, t * per), a1 = min(V, a0 + per);
      for (int i = a0; i < a1; ++i) {
        const double w = share(i);
        if (w == 0.0) continue;
        tok = i;
        wt = w;
        c += w;
        if (c > goal) break;
      }
      if (c > goal) break;
    }
    p.token[b] = tok;
    p.logprob[b] = (float)log(wt / z);
  }
}

}  // namespace
}  // namespace wkvm

extern "C" int wkvm_sample_tokens(const void* logits, int64_t row_stride, const float* u,
                                  const float* temperature, const int32_t* top_k,
                                  const float* top_p, const float* min_p, float temperature0,
                                  int32_t top_k0, float top_p0, float min_p0, int64_t* tokens,
                                  float* logprobs, int32_t B, int32_t V, int32_t dtype,
                                  int32_t* status, wkvm_stream_t stream) {
  if (B < 0 || V <= 0) return WKVM_ERR_INVALID_ARG;
  if (dtype != WKVM_DTYPE_F32 && dtype != WKVM_DTYPE_BF16 && dtype != WKVM_DTYPE_F16)
    return WKVM_ERR_DTYPE;
  if (B == 0) return WKVM_OK;
  if (!logits || !u || !tokens || !logprobs) return WKVM_ERR_INVALID_ARG;
  wkvm::SampleArgs a{logits, row_stride, u, temperature, top_p, min_p, top_k, temperature0,
                     top_p0, min_p0, top_k0, tokens, logprobs, B, V, status};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case WKVM_DTYPE_F32: wkvm::sample_kernel<float><<<B, wkvm::kThreads, 0, st>>>(a); break;
    case WKVM_DTYPE_BF16: wkvm::sample_kernel<__nv_bfloat16><<<B, wkvm::kThreads, 0, st>>>(a); break;
    default: wkvm::sample_kernel<__half><<<B, wkvm::kThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}
