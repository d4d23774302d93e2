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
// each, so HBM bounds it. One thread owns 16 bytes of channels and keeps the
// window in registers.
//
// The launch has two kinds of blocks. Sequence blocks compute the first
// W - 1 outputs of a sequence (those that need the state row) and then write
// its new row; nobody else touches a state row, so the update in place needs
// no second launch and no order between blocks. Tile blocks compute every
// other output from the inputs alone, kTile tokens each, wherever sequences
// begin and end inside the tile.
#include "ssm_common.cuh"

namespace wkvm {
namespace {

constexpr int kTile = 16;     // tokens of a tile block: the window's re-read is (W-1)/16
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

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T e[V]; };

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  const Vec<T, V> u = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32(u.e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  Vec<T, V> u;
#pragma unroll
  for (int i = 0; i < V; ++i) u.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = u;
}

template <typename T, int V, int W, bool SILU>
__global__ void __launch_bounds__(kThreads) short_conv_kernel(ConvArgs p) {
  const int DV = p.D / V;
  const T* wp = static_cast<const T*>(p.w);
  const T* xp = static_cast<const T*>(p.x.p);
  T* op = static_cast<T*>(p.o);
  float w[W][V], bias[V], win[W][V];  // win: the window, oldest first

  auto load_weights = [&](int c) {
    const T* src = wp + (int64_t)c * W;  // channel-major: V * W contiguous weights
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float t[V];
      load_vec<T, V>(src + j * V, t);
#pragma unroll
      for (int i = 0; i < V; ++i) w[(j * V + i) % W][(j * V + i) / W] = t[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = 0.f;
    if (p.bias) load_vec<T, V>(static_cast<const T*>(p.bias) + c, bias);
  };
  auto emit = [&](int64_t token, int c) {
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a = bias[i];
#pragma unroll
      for (int j = 0; j < W; ++j) a = fmaf(w[j][i], win[j][i], a);
      y[i] = SILU ? silu<sizeof(T) == 4>(a) : a;
    }
    store_vec<T, V>(op + token * p.D + c, y);
  };
  auto shift = [&]() {
#pragma unroll
    for (int j = 0; j + 1 < W; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) win[j][i] = win[j + 1][i];
  };

  if ((int)blockIdx.x < p.seq_blocks) {
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
    load_weights(c);
    const int64_t srow = row * (W - 1) * p.D + c;
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) {  // win[1..W-1] <- the state row
#pragma unroll
      for (int i = 0; i < V; ++i) win[j + 1][i] = 0.f;
      if (p.s_in) load_vec<T, V>(static_cast<const T*>(p.s_in) + srow + (int64_t)j * p.D, win[j + 1]);
    }
    const T* xs = xp + act_row(p.seqs, p.x, n, sp.bos) + c;
    const int64_t head = sp.len < p.head ? sp.len : p.head;
    for (int64_t t = 0; t < head; ++t) {
      shift();
      load_vec<T, V>(xs + t * p.x.ts, win[W - 1]);
      emit(sp.bos + t, c);
    }
    if (p.s_out) {
      if (head < sp.len) {  // the last W - 1 inputs lie past the head
#pragma unroll
        for (int j = 0; j + 1 < W; ++j) {
          const int64_t t = sp.len - (W - 1) + j;  // >= 0: head >= W - 1
          load_vec<T, V>(xs + t * p.x.ts, win[j + 1]);
        }
      }
#pragma unroll
      for (int j = 0; j + 1 < W; ++j)
        store_vec<T, V>(static_cast<T*>(p.s_out) + srow + (int64_t)j * p.D, win[j + 1]);
    }
    return;
  }

  // ---- tile block: tokens [t0, t1) of the flattened axis, one channel slice
  const int cblocks = (DV + kThreads - 1) / kThreads;
  const int64_t blk = (int64_t)blockIdx.x - p.seq_blocks;
  const int64_t t0 = blk / cblocks * kTile;
  const int c = ((int)(blk % cblocks) * kThreads + threadIdx.x) * V;
  const int64_t total = p.seqs.cu ? p.seqs.T : (int64_t)p.seqs.nseq * p.seqs.T;
  const int64_t t1 = t0 + kTile < total ? t0 + kTile : total;
  // first sequence that ends past t0, found by the whole warp
  int n = 0;
  if (p.seqs.cu) {
    for (int i = threadIdx.x & 31; i < p.seqs.nseq; i += 32) n += p.seqs.cu[i + 1] <= t0;
    n = __reduce_add_sync(0xffffffffu, n);
  } else {
    n = (int)(t0 / p.seqs.T);
  }
  if (c >= p.D) return;
  load_weights(c);
  for (; n < p.seqs.nseq; ++n) {
    const SeqSpan sp = seq_span(p.seqs, n);
    if (sp.bos >= t1) break;
    int64_t row;
    if (!sp.ok || !state_row(p.ids, p.num_slots, n, &row)) continue;
    int64_t t = t0 - sp.bos > p.head ? t0 - sp.bos : p.head;  // tokens of the sequence
    const int64_t te = t1 - sp.bos < sp.len ? t1 - sp.bos : sp.len;
    if (t >= te) continue;
    const T* xs = xp + act_row(p.seqs, p.x, n, sp.bos) + c;
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) load_vec<T, V>(xs + (t - (W - 1) + j) * p.x.ts, win[j + 1]);
    for (; t < te; ++t) {
      shift();
      load_vec<T, V>(xs + t * p.x.ts, win[W - 1]);
      emit(sp.bos + t, c);
    }
  }
}

template <typename T, int V, int W>
int launch_conv_w(ConvArgs a, bool silu, cudaStream_t st) {
  const int64_t DV = a.D / V;
  const int64_t total = a.seqs.cu ? a.seqs.T : (int64_t)a.seqs.nseq * a.seqs.T;
  // Short rows (a decode step) run wholly in the sequence blocks: no tile
  // blocks to launch, and the inputs are read once. Past kTile tokens a
  // sequence block would be a serial walk, so it keeps the first W - 1 only.
  const bool tiles = a.seqs.cu ? true : a.seqs.T > kTile;
  a.head = tiles ? W - 1 : a.seqs.T;
  const int64_t sb = ((int64_t)a.seqs.nseq * DV + kThreads - 1) / kThreads;
  const int64_t tb = tiles ? (total + kTile - 1) / kTile * ((DV + kThreads - 1) / kThreads) : 0;
  if (sb + tb > INT32_MAX) return WKVM_ERR_SHAPE;
  a.seq_blocks = (int32_t)sb;
  if (silu)
    short_conv_kernel<T, V, W, true><<<(unsigned)(sb + tb), kThreads, 0, st>>>(a);
  else
    short_conv_kernel<T, V, W, false><<<(unsigned)(sb + tb), kThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

template <typename T, int V>
int launch_conv_v(const ConvArgs& a, int W, bool silu, cudaStream_t st) {
  switch (W) {
    case 2: return launch_conv_w<T, V, 2>(a, silu, st);
    case 3: return launch_conv_w<T, V, 3>(a, silu, st);
    case 4: return launch_conv_w<T, V, 4>(a, silu, st);
    default: return WKVM_ERR_SHAPE;
  }
}

template <typename T>
int launch_conv(const ConvArgs& a, int W, bool silu, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  // 16-byte accesses when every row starts on 16 bytes, else one channel a
  // thread (odd channel counts, views at odd offsets)
  const bool vec = a.D % V == 0 && a.x.bs % V == 0 && a.x.ts % V == 0 && aligned_to(a.x.p, 16) &&
                   aligned_to(a.w, 16) && aligned_to(a.bias, 16) && aligned_to(a.o, 16) &&
                   aligned_to(a.s_in, 16) && aligned_to(a.s_out, 16);
  return vec ? launch_conv_v<T, V>(a, W, silu, st) : launch_conv_v<T, 1>(a, W, silu, st);
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
