// Short causal convolution over channels-last activations, with the last
// W - 1 inputs of every sequence kept in a state row [W-1, D] (oldest first):
//
//   y[t][d] = act(bias[d] + sum_j w[d][j] x[t - W + 1 + j][d]),  j < W
//
// where tokens before the sequence's first come from its state row, and the
// row then holds the sequence's own last W - 1 inputs. This is the input
// convolution of selective state space layers and of gated-delta-rule layers.
//
// Streaming: every input is read once, every output written once, 2 W FLOPs
// each, so HBM bounds it: sixteen packed prompts of 32768 x 4096 bf16 take 118
// us, 4.6 TB/s or 70 % of the measured copy rate (218 us with one input in
// flight a thread and scalar arithmetic). One thread owns a few neighbouring channels and keeps
// their weights and window in registers, two channels to a pair.
//
// A sequence's first W - 1 outputs need its state row, which the call also
// replaces. Sequence blocks do both, so nobody else touches a state row: the
// update in place needs no second launch and no order between blocks. Every
// other output needs inputs alone and belongs to a tile block, kTile tokens
// each, wherever sequences begin and end inside the tile. Short rows (a decode
// step) run in sequence blocks alone.
#include "ssm_common.cuh"

namespace wkvm {
namespace {

constexpr int kTile = 32;     // tokens of a tile block: the window's re-read is (W-1)/32
constexpr int kFly = 8;       // inputs of a tile in flight a thread
constexpr int kThreads = 128;

struct ConvArgs {
  Act x;
  const void* w;     // [D, W]
  const void* bias;  // [D] or null
  void* o;           // [tokens, D]
  const void* s_in;  // state rows [.., W-1, D]; null: zeros
  void* s_out;       // null: not wanted
  const int32_t* ids;
  int64_t num_slots;
  Seqs seqs;
  int32_t D;
  int32_t seq_blocks;  // leading blocks that run sequences; the rest run tiles
  int32_t head;        // outputs of a sequence computed by its sequence block
  int* status;
};

// Arithmetic of a lane: two channels in a register pair, or one.
template <int V> using Pair = std::conditional_t<(V > 1), f32x2, float>;
__device__ __forceinline__ f32x2 fma_(f32x2 a, f32x2 b, f32x2 c) { return fma2(a, b, c); }
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }

template <bool EXACT>
__device__ __forceinline__ float silu_of(float x) { return silu<EXACT>(x); }
template <bool EXACT>
__device__ __forceinline__ f32x2 silu_of(f32x2 x) {
  if constexpr (EXACT) {
    const float2 v = unpack2(x);
    return pack2(silu<true>(v.x), silu<true>(v.y));
  } else {
    const float2 t = unpack2(mul2(x, pack2(-kLog2e, -kLog2e)));
    const float2 d = unpack2(add2(pack2(ex2(t.x), ex2(t.y)), pack2(1.f, 1.f)));
    return mul2(x, pack2(rcp(d.x), rcp(d.y)));
  }
}

template <typename T, int V>
__device__ __forceinline__ void widen(const Raw<T, V>& r, Pair<V> (&v)[(V + 1) / 2]) {
  if constexpr (V == 1) {
    v[0] = r.f32(0);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) v[i] = pack2(r.f32(2 * i), r.f32(2 * i + 1));
  }
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
  Raw<T, V> r;
  if constexpr (Raw<T, V>::kBytes == 2)
    r.w[0] = *reinterpret_cast<const uint16_t*>(p);
  else
    move<T, V>(&r, reinterpret_cast<const Raw<T, V>*>(p));
  return r;
}

template <typename T, int V, int W, bool SILU, bool TILES>
__global__ void __launch_bounds__(kThreads) short_conv_kernel(ConvArgs p) {
  constexpr int P = (V + 1) / 2;
  const int DV = p.D / V;
  const T* wp = static_cast<const T*>(p.w);
  const T* xp = static_cast<const T*>(p.x.p);
  T* op = static_cast<T*>(p.o);
  Pair<V> w[W][P], win[W][P];  // win: the window, oldest first
  Raw<T, V> wr[W], br;         // weights and bias as they lie in memory

  // pair (or channel) i of the weights of tap j: V * W weights, channel-major
  auto weight = [&](int j, int i) -> Pair<V> {
    auto at = [&](int c) { return wr[(c * W + j) / V].f32((c * W + j) % V); };
    if constexpr (V == 1) return at(0);
    else return pack2(at(2 * i), at(2 * i + 1));
  };
  auto load_weights = [&](int c) {
    const T* src = wp + (int64_t)c * W;
#pragma unroll
    for (int j = 0; j < W; ++j) wr[j] = load_raw<T, V>(src + j * V);
#pragma unroll
    for (int i = 0; i < Raw<T, V>::kWords; ++i) br.w[i] = 0;
    if (p.bias) br = load_raw<T, V>(static_cast<const T*>(p.bias) + c);
    if constexpr (TILES) {  // used again and again: widened once
#pragma unroll
      for (int j = 0; j < W; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) w[j][i] = weight(j, i);
    }
  };
  auto put = [&](T* dst, const Pair<V> (&y)[P]) {
    if constexpr (V == 1) {
      *dst = from_f32<T>(y[0]);
    } else {
      Raw<T, V> out;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 v = unpack2(y[i]);
        out.set2(2 * i, v.x, v.y);
      }
      move<T, V>(reinterpret_cast<Raw<T, V>*>(dst), &out);
    }
  };
  auto emit = [&](int64_t token, int c) {
    Pair<V> y[P];
    widen<T, V>(br, y);
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
      for (int j = 0; j < W; ++j) y[i] = fma_(TILES ? w[j][i] : weight(j, i), win[j][i], y[i]);
      if (SILU) y[i] = silu_of<sizeof(T) == 4>(y[i]);
    }
    put(op + token * p.D + c, y);
  };
  auto shift = [&](const Raw<T, V>& in) {
#pragma unroll
    for (int j = 0; j + 1 < W; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) win[j][i] = win[j + 1][i];
    widen<T, V>(in, win[W - 1]);
  };

  if (!TILES || (int)blockIdx.x < p.seq_blocks) {
    const int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (e >= (int64_t)p.seqs.nseq * DV) return;
    const int n = (int)(e / DV), c = (int)(e - (int64_t)n * DV) * V;
    int64_t row;
    const SeqSpan sp = seq_span(p.seqs, n);
    if (!state_row(p.ids, p.num_slots, n, &row)) {
      if (c == 0) report(p.status, WKVM_ERR_SLOT_RANGE);
      return;
    }
    if (!sp.ok) {
      if (c == 0) report(p.status, WKVM_ERR_INVALID_ARG);
      return;
    }
    const int64_t srow = row * (W - 1) * p.D + c;
    const T* xs = xp + act_row(p.seqs, p.x, n, sp.bos) + c;
    const int64_t head = sp.len < p.head ? sp.len : p.head;
    Raw<T, V> next;
    if (head > 0) next = load_raw<T, V>(xs);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) {  // win[1..W-1] <- the state row
#pragma unroll
      for (int i = 0; i < P; ++i) win[j + 1][i] = 0;
      if (p.s_in) widen<T, V>(load_raw<T, V>(static_cast<const T*>(p.s_in) + srow + (int64_t)j * p.D), win[j + 1]);
    }
    load_weights(c);
    for (int64_t t = 0; t < head; ++t) {
      shift(next);
      if (t + 1 < head) next = load_raw<T, V>(xs + (t + 1) * p.x.ts);
      emit(sp.bos + t, c);
    }
    if (p.s_out) {
      // the last W - 1 inputs: those in the window, unless the sequence goes on
      // in tile blocks
#pragma unroll
      for (int j = 0; j + 1 < W; ++j) {
        if (head < sp.len) widen<T, V>(load_raw<T, V>(xs + (sp.len - (W - 1) + j) * p.x.ts), win[j + 1]);
        put(static_cast<T*>(p.s_out) + srow + (int64_t)j * p.D, win[j + 1]);
      }
    }
    return;
  }
  if constexpr (!TILES) return;

  // ---- tile block: tokens [t0, t1) of the flattened axis, one channel slice
  const int cblocks = (DV + kThreads - 1) / kThreads;
  const int64_t blk = (int64_t)blockIdx.x - p.seq_blocks;
  const int64_t t0 = blk / cblocks * kTile;
  const int c = ((int)(blk % cblocks) * kThreads + threadIdx.x) * V;
  const int64_t total = p.seqs.cu ? p.seqs.T : (int64_t)p.seqs.nseq * p.seqs.T;
  const int64_t t1 = t0 + kTile < total ? t0 + kTile : total;
  // the first sequence that ends past t0 and the last that begins before t1,
  // found by the whole warp; offsets that descend leave others between them,
  // which the loop skips
  int n = 0, last = 0;
  if (p.seqs.cu) {
    n = p.seqs.nseq;
    for (int i = threadIdx.x & 31; i < p.seqs.nseq; i += 32) {
      if (p.seqs.cu[i + 1] > t0) n = min(n, i);
      if (p.seqs.cu[i] < t1) last = i;
    }
    n = __reduce_min_sync(0xffffffffu, n);
    last = __reduce_max_sync(0xffffffffu, last);
  } else {
    n = (int)(t0 / p.seqs.T);
    last = (int)((t1 - 1) / p.seqs.T);
  }
  if (c >= p.D) return;
  load_weights(c);
  for (; n <= last; ++n) {
    const SeqSpan sp = seq_span(p.seqs, n);
    int64_t row;
    if (!sp.ok || !state_row(p.ids, p.num_slots, n, &row)) continue;
    const int64_t ta = t0 - sp.bos > p.head ? t0 - sp.bos : p.head;  // tokens of the sequence
    const int64_t te = t1 - sp.bos < sp.len ? t1 - sp.bos : sp.len;
    if (ta >= te) continue;
    const T* xs = xp + act_row(p.seqs, p.x, n, sp.bos) + c + ta * p.x.ts;
    const int64_t token = sp.bos + ta;
    const int many = (int)(te - ta);
    Raw<T, V> in[kFly];
#pragma unroll
    for (int f = 0; f < kFly; ++f)
      if (f < many) in[f] = load_raw<T, V>(xs + f * p.x.ts);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) widen<T, V>(load_raw<T, V>(xs + (j - (W - 1)) * p.x.ts), win[j + 1]);
    for (int t = 0; t < many; t += kFly) {
#pragma unroll
      for (int f = 0; f < kFly; ++f) {
        if (t + f >= many) break;
        shift(in[f]);
        if (t + f + kFly < many) in[f] = load_raw<T, V>(xs + (int64_t)(t + f + kFly) * p.x.ts);
        emit(token + t + f, c);
      }
    }
  }
}

template <typename T, int V, int W, bool TILES>
int launch_conv_w(ConvArgs a, bool silu, cudaStream_t st) {
  const int64_t DV = a.D / V;
  const int64_t total = a.seqs.cu ? a.seqs.T : (int64_t)a.seqs.nseq * a.seqs.T;
  a.head = TILES ? W - 1 : a.seqs.T;
  const int64_t sb = ((int64_t)a.seqs.nseq * DV + kThreads - 1) / kThreads;
  const int64_t tb = TILES ? (total + kTile - 1) / kTile * ((DV + kThreads - 1) / kThreads) : 0;
  if (sb + tb > INT32_MAX) return WKVM_ERR_SHAPE;
  a.seq_blocks = (int32_t)sb;
  const auto kern = silu ? short_conv_kernel<T, V, W, true, TILES> : short_conv_kernel<T, V, W, false, TILES>;
  kern<<<(unsigned)(sb + tb), kThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

template <typename T, int V, bool TILES>
int launch_conv_v(const ConvArgs& a, int W, bool silu, cudaStream_t st) {
  switch (W) {
    case 2: return launch_conv_w<T, V, 2, TILES>(a, silu, st);
    case 3: return launch_conv_w<T, V, 3, TILES>(a, silu, st);
    case 4: return launch_conv_w<T, V, 4, TILES>(a, silu, st);
    default: return WKVM_ERR_SHAPE;
  }
}

template <typename T>
int launch_conv(const ConvArgs& a, int W, bool silu, cudaStream_t st) {
  // Whole-vector accesses when every row starts on the vector's size, else one
  // channel a thread (odd channel counts, views at odd offsets). A sequence
  // block keeps 16 bytes of channels a thread; in a tile, eight 16-bit channels
  // and their inputs in flight would take 140 registers, so four.
  constexpr int VS = 16 / sizeof(T), VT = 4;
  auto fits = [&](int v) {
    const uintptr_t n = v * sizeof(T);
    return a.D % v == 0 && a.x.bs % v == 0 && a.x.ts % v == 0 && aligned_to(a.x.p, n) && aligned_to(a.w, n) &&
           aligned_to(a.bias, n) && aligned_to(a.o, n) && aligned_to(a.s_in, n) && aligned_to(a.s_out, n);
  };
  // Past kTile tokens a sequence block would be a serial walk, so it keeps the
  // first W - 1 only; shorter rows need no tile blocks.
  if (!a.seqs.cu && a.seqs.T <= kTile)
    return fits(VS) ? launch_conv_v<T, VS, false>(a, W, silu, st) : launch_conv_v<T, 1, false>(a, W, silu, st);
  return fits(VT) ? launch_conv_v<T, VT, true>(a, W, silu, st) : launch_conv_v<T, 1, true>(a, W, silu, st);
}

int run_conv(ConvArgs a, int W, int act, int dtype, cudaStream_t st) {
  a.x = plain_strides(a.x, a.seqs);
  if (a.seqs.nseq < 0 || a.seqs.T < 0 || a.D <= 0) return WKVM_ERR_INVALID_ARG;
  if (act != WKVM_ACT_NONE && act != WKVM_ACT_SILU) return WKVM_ERR_INVALID_ARG;
  if (W < 2 || W > 4) return WKVM_ERR_SHAPE;
  if (dtype != WKVM_DTYPE_F32 && dtype != WKVM_DTYPE_BF16 && dtype != WKVM_DTYPE_F16)
    return WKVM_ERR_DTYPE;
  if (a.seqs.nseq == 0) return WKVM_OK;
  if (!a.w || (a.seqs.T > 0 && (!a.x.p || !a.o))) return WKVM_ERR_INVALID_ARG;
  switch (dtype) {
    case WKVM_DTYPE_F32: return launch_conv<float>(a, W, act == WKVM_ACT_SILU, st);
    case WKVM_DTYPE_BF16: return launch_conv<__nv_bfloat16>(a, W, act == WKVM_ACT_SILU, st);
    default: return launch_conv<__half>(a, W, act == WKVM_ACT_SILU, st);
  }
}

}  // namespace
}  // namespace wkvm

extern "C" int wkvm_short_conv(const void* x, int64_t x_batch_stride, int64_t x_token_stride,
                               const void* weight, const void* bias, void* o, const void* s0,
                               void* st, const int64_t* cu_seqlens, int32_t B, int32_t T,
                               int32_t D, int32_t W, int32_t activation, int32_t dtype,
                               int32_t* status, wkvm_stream_t stream) {
  wkvm::ConvArgs a{{x, x_batch_stride, x_token_stride}, weight, bias, o, s0, st, nullptr, 0,
                   {cu_seqlens, B, T}, D, 0, 0, status};
  return wkvm::run_conv(a, W, activation, dtype, (cudaStream_t)stream);
}

extern "C" int wkvm_short_conv_slots(const void* x, int64_t x_batch_stride,
                                     int64_t x_token_stride, const void* weight, const void* bias,
                                     void* o, void* bank_layer, int64_t num_slots,
                                     const int32_t* slot_ids, const int64_t* cu_seqlens, int32_t B,
                                     int32_t T, int32_t D, int32_t W, int32_t activation,
                                     int32_t dtype, int32_t* status, wkvm_stream_t stream) {
  if (B > 0 && (!bank_layer || !slot_ids || num_slots <= 0)) return WKVM_ERR_INVALID_ARG;
  wkvm::ConvArgs a{{x, x_batch_stride, x_token_stride}, weight, bias, o, bank_layer, bank_layer,
                   slot_ids, num_slots, {cu_seqlens, B, T}, D, 0, 0, status};
  return wkvm::run_conv(a, W, activation, dtype, (cudaStream_t)stream);
}
