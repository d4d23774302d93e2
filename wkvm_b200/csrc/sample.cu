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
// Masses: where one token ends and the next begins moves by the error of a
// running mass, and with 65,536 tokens an error of 1e-7 would change about
// one row's token in two hundred. So weights are fp64 (2e-13), rounded once
// to units of 2^-s and summed as 64-bit integers: sums are exact, whatever
// the order, so atomics and every split over threads give the same result.
// s is as large as V weights of 1 allow (46 for 65,536 logits): the rounding
// moves a mass by V 2^-(s+1) at most, 2^-31 of the largest weight there.
//
// All three filters keep a prefix of the descending order, so what is kept is
// one logit and a bound on the ids that equal it. A row's CTAs (a cluster for
// large vocabularies and few rows) find that bound by histograms
// of counts (top-k) or masses (top-p) over the logits above a lower bound,
// then finish on a sorted list of at most kCap candidates in one CTA. Only a
// larger set is narrowed by further histograms and drawn from by a pass over
// the whole row. HBM is read once: later passes find the slice in shared
// memory, or, in vocabularies too long for sixteen CTAs', in L2. At 256 rows of
// 65,536 fp32 logits (10 us of HBM), on the device: 25 us greedy, 63 top-k and
// top-p, 65 without a filter, 170 top-p 0.8 to 0.99 (thousands of tokens kept),
// which evaluates the weights twice; 90 with a mix of settings. The issue of
// some ninety instructions a logit bounds it, then the latency of one row's
// phases (one row: 13 us top-k, 21 top-p).
#include <cooperative_groups.h>
#include <float.h>

#include "common.cuh"

namespace wkvm {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

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
  int32_t V;
  int32_t slice;  // logits of one CTA, a multiple of kNT
  int32_t ctas;   // of a row
  double shift;   // 2^(52-s): adding it leaves a weight's units in the low bits
  bool vec;       // rows start on 16 bytes
};

constexpr int kNT = 512, kWarps = kNT / 32;
constexpr int kBins = 1024;
constexpr int kCap = 1024;        // candidates one CTA sorts
constexpr int kRankSort = 384;    // of which so many by counting
constexpr int kGroups = 10;       // 1, 2, 4, .. 512 sets of a CTA's threads
constexpr int kMaxCtas = 16;      // CTAs of a row (16: a cluster size that a kernel has to ask for)
constexpr int kSmemSlice = 16384; // logits of a slice kept in shared memory (two CTAs an SM)

// Ascending unsigned order of floats; -0 counts as 0, -inf and NaN as 0u.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// 2^t for -1000 < t <= 0, to 1e-13: with k = t rounded to 1/64 and r the rest,
// 2^(k >> 6) times table[k & 63] = 2^((k & 63) / 64) times 1 + r p(r), the
// power series of e^(r ln 2) to degree 4 (|r ln 2| < 0.0055).
__device__ __forceinline__ double exp2_neg(double t, const double* table) {
  const double magic = 105553116266496.0;  // 1.5 * 2^46: rounds to 1/64
  const double u = t + magic;
  const int k = __double2loint(u);
  const double r = t - (u - magic);
  double p = 0.009618129107628477;
  p = fma(p, r, 0.05550410866482158);
  p = fma(p, r, 0.24022650695910072);
  p = fma(p, r, 0.6931471805599453);
  const double e = table[k & 63];
  const double w = fma(e, r * p, e);
  return __hiloint2double(__double2hiint(w) + ((k >> 6) << 20), __double2loint(w));
}

// The next smaller double of a positive one.
__device__ __forceinline__ double below(double x) { return __longlong_as_double(__double_as_longlong(x) - 1); }

struct Found {          // what a level of a selection found, the same in every CTA
  int bin;              // the bin with the boundary; -1: everything is kept
  uint32_t above, in;   // candidates in the bins above it, and in it
  u64 mass_above, mass_in;
};

// Shared memory of a CTA ahead of its slice of logits. Fields named peer_* are
// written by the other CTAs of the cluster, [rank] by rank.
struct alignas(16) Shared {
  union {
    struct {                          // histogram: counts, and masses in two words
      uint32_t cnt[kBins], mass_lo[kBins], mass_hi[kBins];
    };
    struct {                          // then candidates: ~key << 32 | id, ascending = the descending order
      u64 list[kCap], weight[kCap];
    };
  };
  double exp2_table[64];            // 2^(i / 64)
  u64 warp_sum[kWarps];
  uint32_t warp_u32[7][kWarps];
  uint32_t peer_max[kMaxCtas], peer_least[kGroups][kMaxCtas];
  uint32_t peer_lo[kMaxCtas], peer_hi[kMaxCtas], peer_cnt[kMaxCtas];
  u64 peer_mass[kMaxCtas], peer_total[kMaxCtas];
  Found found;
  uint32_t n_list;
  float tau;                        // the last kept logit
  int32_t limit;                    // ids below it are kept among its equals
  int32_t first;                    // greedy
  int32_t owner;                    // the warp whose block holds the drawn token
};

static_assert(sizeof(Shared) % 16 == 0, "the slice behind it is read 16 bytes at a time");

template <typename T, bool SMEM>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  Shared* s;
  const float* vals;  // SMEM: the slice
  const T* row;       // the slice in global memory
  bool vec;           // it starts on 16 bytes
  int rank, ctas, tid, lane, warp, slice, base;  // base: the slice's first id
  int n;              // logits of the slice that exist
  float top;         // the row's maximum
  bool flat;         // it is +inf: only logits equal to it are kept, all of weight 1
  double c;          // log2(e) / temperature
  double shift;      // of units(), a power of two >= 1
  // kept: l > tau, or l == tau and id < limit (NaN and -inf never are)
  float tau;
  int32_t limit;

  // Weights of four kept logits (others give any value). Four at once: each is
  // a chain of dependent fp64 operations, and only other chains fill its latency.
  template <int W>
  __device__ __forceinline__ void weights(const float (&l)[W], double (&w)[W]) const {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const double t = ((double)l[j] - (double)top) * c;
      // t <= 0, at least about -60: that is no unit any more. Negative numbers
      // ascend with their bits, so the upper word's smaller one is taken.
      const uint32_t hi = min((uint32_t)__double2hiint(t), 0xc04e0000u);
      w[j] = flat ? 1.0 : exp2_neg(__hiloint2double((int)hi, __double2loint(t)), s->exp2_table);
    }
  }
  __device__ __forceinline__ double weight(float l) const {
    const float a[1] = {l};
    double w[1];
    weights<1>(a, w);
    return w[0];
  }
  __device__ u64 units(double w) const {
    const double x = w + shift;
    return (u64)(uint32_t)(__double2hiint(x) - __double2hiint(shift)) << 32 | (uint32_t)__double2loint(x);
  }
  __device__ double weight_of(u64 z) const { return (double)z * (shift * 0x1p-52); }
  __device__ __forceinline__ bool kept(float l, int id) const { return l > tau || (l == tau && id < limit); }

  __device__ float at(int i) const {
    if constexpr (SMEM) return vals[i];
    return i < n ? to_f32(row[i]) : -INFINITY;
  }
  // f(logits, i) for the logits [i0, i1) four at a time, i the first one's
  // index, dealt to `nt` threads of which this is thread t. Past the slice's
  // end they read as -inf. i0 and i1 are multiples of 8.
  template <typename F>
  __device__ __forceinline__ void each(int i0, int i1, int t, int nt, F f) const {
    if constexpr (SMEM) {
      for (int i = i0 + t * 4; i < i1; i += nt * 4) {
        const float4 v = *reinterpret_cast<const float4*>(vals + i);
        const float l[4] = {v.x, v.y, v.z, v.w};
        f(l, i);
      }
    } else {
      const int whole = vec ? min(i1, max(i0, n / kVec * kVec)) : i0;
      uint4 next = make_uint4(0, 0, 0, 0);
      int i = i0 + t * kVec;
      if (i < whole) next = *reinterpret_cast<const uint4*>(row + i);
      for (; i < whole; i += nt * kVec) {
        const uint4 q = next;
        if (i + nt * kVec < whole) next = *reinterpret_cast<const uint4*>(row + i + nt * kVec);
#pragma unroll
        for (int h = 0; h < kVec; h += 4) {
          float l[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) l[j] = to_f32(reinterpret_cast<const T*>(&q)[h + j]);
          f(l, i + h);
        }
      }
      for (int i = whole + t * 4; i < min(i1, n); i += nt * 4) {
        float l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) l[j] = at(i + j);
        f(l, i);
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const { each(0, slice, tid, kNT, f); }

  template <typename X>
  __device__ X warp_add(X x) const {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
  }
  // Sum over the CTA, returned to every thread.
  __device__ u64 block_add(u64 x) const {
    x = warp_add(x);
    __syncthreads();
    if (lane == 0) s->warp_sum[warp] = x;
    __syncthreads();
    u64 t = 0;
    for (int i = 0; i < kWarps; ++i) t += s->warp_sum[i];
    return t;
  }
  // Another CTA's shared memory may be touched only once that CTA is known to
  // run: behind wait_started(), or any sync(). Every thread arrives at the
  // kernel's entry, so that loading the slice hides the wait.
  __device__ void arrive_started() const {
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  }
  __device__ void wait_started() const {
    if (ctas > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
  }
  __device__ Shared* peer(int r) const { return ctas == 1 ? s : cg::this_cluster().map_shared_rank(s, r); }
  __device__ void sync() const {  // the row's CTAs
    if (ctas == 1) __syncthreads(); else cg::this_cluster().sync();
  }
};

// A level's bins: logits [lo, hi] into kBins bins, the largest first. Linear
// in the logit where that is safe, else in the key; any monotone map does.
struct Bins {
  float lo, hi, scale;  // scale 0: linear in the key
  u64 step;             // 2^32 bins / keys
  __device__ Bins(float l, float h) : lo(l), hi(h), scale(0.f), step(0) {
    const float range = hi - lo;
    if (range > 1e-30f && range < 1e30f)
      scale = kBins / range;
    else
      step = ((u64)kBins << 32) / ((u64)(key_of(hi) - key_of(lo)) + 1);
  }
  __device__ __forceinline__ bool holds(float l) const { return l >= lo && l <= hi; }
  __device__ __forceinline__ int operator()(float l) const {
    const int b = scale > 0.f ? (int)((hi - l) * scale) : (int)(((u64)(key_of(hi) - key_of(l)) * step) >> 32);
    return b < kBins - 1 ? b : kBins - 1;
  }
};

// One level: histogram of the kept candidates in [b.lo, b.hi], and
// the first bin at which above + the running count (or mass) reaches the goal.
// `rest`: mass of what is kept below b.lo joins the total, and the goal is
// share times that total (first level of top-p). Two cluster barriers.
template <bool MASS, typename R>
__device__ void level(R& r, const Bins& b, uint32_t above, u64 mass_above, double goal, bool rest,
                      double share, u64* total) {
  Shared* s = r.s;
  for (int i = r.tid; i < kBins; i += kNT) {
    s->cnt[i] = 0;
    if (MASS) s->mass_lo[i] = s->mass_hi[i] = 0;
  }
  __syncthreads();
  u64 all = 0;
  r.each([&](const float (&l)[4], int i) {
    bool in[4], any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) any |= in[j] = l[j] <= b.hi && (rest || l[j] >= b.lo) && r.kept(l[j], r.base + i + j);
    if (!any) return;
    double w[4];
    if (MASS) r.weights(l, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!in[j]) continue;
      u64 m = 0;
      if (MASS) m = r.units(w[j]);
      if (MASS && rest) all += m;
      if (l[j] < b.lo) continue;
      const int bin = b(l[j]);
      atomicAdd(&s->cnt[bin], 1u);
      if (MASS) {
        const uint32_t lo = (uint32_t)m, old = atomicAdd(&s->mass_lo[bin], lo);
        const uint32_t hi = (uint32_t)(m >> 32) + (old + lo < old);
        if (hi) atomicAdd(&s->mass_hi[bin], hi);
      }
    }
  });
  if (MASS && rest) {
    all = r.block_add(all);
    if (r.tid < r.ctas) r.peer(r.tid)->peer_total[r.rank] = all;
  }
  r.sync();
  if (MASS && rest) {
    all = 0;
    for (int i = 0; i < r.ctas; ++i) all += s->peer_total[i];
    *total = all;
    goal = share * (double)all;
  }
  if (r.rank == 0) {
    // two neighbouring bins a thread, summed over the cluster
    uint32_t c[2] = {0, 0};
    u64 m[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < kMaxCtas; ++p) {  // every peer's bins in flight at once
      if (p >= r.ctas) break;
      const Shared* o = r.peer(p);
      const uint2 n = *reinterpret_cast<const uint2*>(&o->cnt[2 * r.tid]);
      c[0] += n.x;
      c[1] += n.y;
      if (MASS) {
        const uint2 lo = *reinterpret_cast<const uint2*>(&o->mass_lo[2 * r.tid]);
        const uint2 hi = *reinterpret_cast<const uint2*>(&o->mass_hi[2 * r.tid]);
        m[0] += (u64)hi.x << 32 | lo.x;
        m[1] += (u64)hi.y << 32 | lo.y;
      }
    }
    uint32_t cs = c[0] + c[1];
    u64 ms = m[0] + m[1];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t cu = __shfl_up_sync(0xffffffffu, cs, off);
      const u64 mu = __shfl_up_sync(0xffffffffu, ms, off);
      if (r.lane >= off) {
        cs += cu;
        ms += mu;
      }
    }
    __syncthreads();
    if (r.lane == 31) {
      s->warp_u32[0][r.warp] = cs;
      s->warp_sum[r.warp] = ms;
    }
    if (r.tid == 0) s->found.bin = -1;
    __syncthreads();
    uint32_t cb = above;
    u64 mb = mass_above;
    for (int i = 0; i < r.warp; ++i) {
      cb += s->warp_u32[0][i];
      mb += s->warp_sum[i];
    }
    cb += cs - c[0] - c[1];  // what is above this thread's bins
    mb += ms - m[0] - m[1];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool before = MASS ? (double)mb < goal : (double)cb < goal;
      const bool reached = MASS ? (double)(mb + m[j]) >= goal : (double)(cb + c[j]) >= goal;
      if (c[j] && before && reached) s->found = {2 * r.tid + j, cb, c[j], mb, m[j]};
      cb += c[j];
      mb += m[j];
    }
    __syncthreads();
    // to every CTA
    const int words = sizeof(Found) / 4;
    for (int i = r.tid; i < words * (r.ctas - 1); i += kNT)
      reinterpret_cast<uint32_t*>(&r.peer(1 + i / words)->found)[i % words] =
          reinterpret_cast<const uint32_t*>(&s->found)[i % words];
    if (r.tid == 0) s->n_list = 0;
  }
  r.sync();
}

// Kept candidates that `take(logit)` names go to the first CTA's list.
template <typename R, typename F>
__device__ void gather(R& r, F take) {
  Shared* first = r.peer(0);
  r.each([&](const float (&l)[4], int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!take(l[j]) || !r.kept(l[j], r.base + i + j)) continue;
      const uint32_t slot = atomicAdd(&first->n_list, 1u);
      if (slot < kCap) first->list[slot] = ((u64)~key_of(l[j]) << 32) | (uint32_t)(r.base + i + j);
    }
  });
  r.sync();
}

// Sorts the first n entries of the list ascending (one CTA, n <= kCap).
__device__ __forceinline__ void sort_list(Shared* s, int tid, int n) {
  if (n <= kRankSort) {
    // few: every entry counts those ahead of it (they differ, by their ids);
    // n reads without a barrier beat some forty steps that each wait
    if (tid == 0) s->list[n] = ~0ull;  // an even number to read
    __syncthreads();
    if (tid < n) {
      const u64 mine = s->list[tid];
      int rank = 0;
#pragma unroll 4
      for (int i = 0; i < n; i += 2) {
        const ulonglong2 e = *reinterpret_cast<const ulonglong2*>(&s->list[i]);
        rank += (e.x < mine) + (e.y < mine);
      }
      s->weight[rank] = mine;
    }
    __syncthreads();
    if (tid < n) s->list[tid] = s->weight[tid];
    __syncthreads();
    return;
  }
  int size = 2;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kNT) s->list[i] = ~0ull;
  __syncthreads();
  // thread t compares the pair at a = 2t with bit j cleared: with j <= 32 a
  // warp's pairs are its own 64 entries, and only wider steps meet the others
  const int t = tid;
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      if (t < size / 2) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const u64 x = s->list[a], y = s->list[b];
        if ((x > y) == ((a & k) == 0)) {
          s->list[a] = y;
          s->list[b] = x;
        }
      }
      if (j > 32 || (j == 1 && k >= 64)) __syncthreads(); else __syncwarp();
    }
  __syncthreads();
}

// Inclusive sums of weight[0, n) in place (one CTA, two neighbours a thread).
__device__ __forceinline__ void scan_weights(Shared* s, int tid, int n) {
  const int i = 2 * tid;
  const u64 a = i < n ? s->weight[i] : 0, b = i + 1 < n ? s->weight[i + 1] : 0;
  u64 x = a + b;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, x, off);
    if ((tid & 31) >= off) x += up;
  }
  __syncthreads();
  if ((tid & 31) == 31) s->warp_sum[(tid >> 5)] = x;
  __syncthreads();
  for (int w = 0; w < (tid >> 5); ++w) x += s->warp_sum[w];
  if (i < n) s->weight[i] = x - b;
  if (i + 1 < n) s->weight[i + 1] = x;
  __syncthreads();
}

__device__ __forceinline__ uint32_t list_key(u64 e) { return ~(uint32_t)(e >> 32); }

// The row's end on the list: n candidates, of which the first k are in play.
// total: the mass top-p takes its share of (0: of these k).
template <typename R>
__device__ void finish_list(R& r, int n, int k, double tp, double mp, double u, u64 total,
                            int64_t* token, float* logprob) {
  Shared* s = r.s;
  sort_list(s, r.tid, n);
  if (k < n) n = k;
  auto weigh = [&](int i) { return r.weight(value_of(list_key(s->list[i]))); };
  if (tp < 1.0) {
    for (int i = r.tid; i < n; i += kNT) s->weight[i] = r.units(weigh(i));
    __syncthreads();
    scan_weights(s, r.tid, n);
    const double goal = tp * (double)(total ? total : s->weight[n - 1]);
    // entry i stays while the mass before it is short of the goal
    uint32_t stay = 0;
    for (int i = r.tid; i < n; i += kNT) stay += i == 0 || (double)s->weight[i - 1] < goal;
    n = (int)r.block_add(stay);
  }
  if (mp > 0.0) {
    uint32_t stay = 0;
    for (int i = r.tid; i < n; i += kNT) stay += i == 0 || weigh(i) >= mp || value_of(list_key(s->list[i])) == r.top;
    n = (int)r.block_add(stay);
  }
  // draw in order of ids
  for (int i = r.tid; i < n; i += kNT) {
    const u64 e = s->list[i];
    s->list[i] = (e << 32) | (e >> 32);
  }
  __syncthreads();
  sort_list(s, r.tid, n);
  auto by_id = [&](int i) { return r.weight(value_of(~(uint32_t)s->list[i])); };
  for (int i = r.tid; i < n; i += kNT) s->weight[i] = r.units(by_id(i));
  __syncthreads();
  scan_weights(s, r.tid, n);
  const u64 z = s->weight[n - 1];
  double goal = u * (double)z;
  if (!(goal < (double)z)) goal = below((double)z);
  for (int i = r.tid; i < n; i += kNT) {
    const u64 before = i ? s->weight[i - 1] : 0;
    if (s->weight[i] > before && (double)s->weight[i] > goal && !((double)before > goal)) {
      *token = (int64_t)(s->list[i] >> 32);
      *logprob = (float)log(by_id(i) / r.weight_of(z));
    }
  }
}

// Keeps, of the kept candidates that equal `tie`, the `want` lowest ids.
template <typename R>
__device__ void limit_ties(R& r, float tie, uint32_t want) {
  Shared* s = r.s;
  const int per = r.slice / kWarps, i0 = r.warp * per;
  uint32_t c = 0;
  r.each(i0, i0 + per, r.lane, 32, [&](const float (&l)[4], int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c += l[j] == tie && r.kept(tie, r.base + i + j);
  });
  c = r.warp_add(c);
  __syncthreads();
  if (r.lane == 0) s->warp_u32[0][r.warp] = c;
  __syncthreads();
  if (r.tid < r.ctas) {
    uint32_t t = 0;
    for (int w = 0; w < kWarps; ++w) t += s->warp_u32[0][w];
    r.peer(r.tid)->peer_cnt[r.rank] = t;
  }
  r.sync();
  uint32_t before = 0;
  for (int p = 0; p < r.rank; ++p) before += s->peer_cnt[p];
  for (int w = 0; w < r.warp; ++w) before += s->warp_u32[0][w];
  if (before < want && before + s->warp_u32[0][r.warp] >= want) {  // one warp of the cluster
    for (int i = i0; i < i0 + per; i += 32) {
      const bool is = r.at(i + r.lane) == tie && r.kept(tie, r.base + i + r.lane);
      const uint32_t b = __ballot_sync(0xffffffffu, is);
      if (before + __popc(b) < want) {
        before += __popc(b);
        continue;
      }
      const bool last = is && before + __popc(b & ((2u << r.lane) - 1)) == want;
      if (last)
        for (int p = 0; p < r.ctas; ++p) r.peer(p)->limit = r.base + i + r.lane + 1;
      break;
    }
  }
  r.sync();
  r.tau = tie;
  r.limit = s->limit;
}

// Narrows what is kept to the first candidates in descending order whose
// count reaches `goal` (or whose mass reaches tp of the mass of all kept).
// Returns true when the row was finished on the list.
template <bool MASS, typename R>
__device__ bool select(R& r, float lo, double goal, int k, double tp, double mp, double u,
                       int64_t* token, float* logprob) {
  Shared* s = r.s;
  Bins b(lo, r.top);
  uint32_t above = 0;
  u64 mass_above = 0, total = 0;
  for (bool first = true;; first = false) {
    level<MASS>(r, b, above, mass_above, goal, MASS && first, tp, &total);
    if (MASS && first) goal = tp * (double)total;
    Found f = s->found;
    // counts: fewer than the goal in all. masses: a goal that no mass is short
    // of (a share of nothing), the top alone is kept
    if (f.bin < 0) {
      if (!MASS) return false;
      limit_ties(r, r.top, 1);
      return false;
    }
    if (f.above + f.in <= kCap) {
      gather(r, [&](float l) { return l > b.hi || (l >= b.lo && b(l) <= f.bin); });
      if (r.rank == 0) finish_list(r, (int)(f.above + f.in), MASS ? INT32_MAX : k, tp, mp, u, total, token, logprob);
      return true;
    }
    if (f.in <= kCap) {
      gather(r, [&](float l) { return b.holds(l) && b(l) == f.bin; });
      if (r.rank == 0) {
        const int n = (int)f.in;
        sort_list(s, r.tid, n);
        for (int i = r.tid; i < n; i += kNT) s->weight[i] = MASS ? r.units(r.weight(value_of(list_key(s->list[i])))) : 1;
        __syncthreads();
        scan_weights(s, r.tid, n);
        const u64 base = MASS ? f.mass_above : f.above;
        for (int i = r.tid; i < n; i += kNT) {
          const double before = (double)(base + (i ? s->weight[i - 1] : 0));
          if (before < goal && ((double)(base + s->weight[i]) >= goal || i == n - 1))
            for (int p = 0; p < r.ctas; ++p) {
              r.peer(p)->tau = value_of(list_key(s->list[i]));
              r.peer(p)->limit = (int32_t)(uint32_t)s->list[i] + 1;
            }
        }
      }
      r.sync();
      r.tau = s->tau;
      r.limit = s->limit;
      return false;
    }
    // too many: their smallest and largest key bound the next level
    uint32_t kl = 0xffffffffu, kh = 0;
    r.each([&](const float (&l)[4], int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!b.holds(l[j]) || !r.kept(l[j], r.base + i + j) || b(l[j]) != f.bin) continue;
        kl = min(kl, key_of(l[j]));
        kh = max(kh, key_of(l[j]));
      }
    });
    kl = __reduce_min_sync(0xffffffffu, kl);
    kh = __reduce_max_sync(0xffffffffu, kh);
    __syncthreads();
    if (r.lane == 0) {
      s->warp_u32[0][r.warp] = kl;
      s->warp_u32[1][r.warp] = kh;
    }
    __syncthreads();
    if (r.tid < r.ctas) {
      for (int w = 0; w < kWarps; ++w) {
        kl = min(kl, s->warp_u32[0][w]);
        kh = max(kh, s->warp_u32[1][w]);
      }
      r.peer(r.tid)->peer_lo[r.rank] = kl;
      r.peer(r.tid)->peer_hi[r.rank] = kh;
    }
    r.sync();
    for (int p = 0; p < r.ctas; ++p) {
      kl = min(kl, s->peer_lo[p]);
      kh = max(kh, s->peer_hi[p]);
    }
    if (kl == kh) {  // equal logits: as many as it takes
      uint32_t want = (uint32_t)(goal - (double)f.above);
      if (MASS) {
        const u64 w = r.units(r.weight(value_of(kl)));
        want = (uint32_t)fmin((goal - (double)f.mass_above) / (double)w, (double)(f.in - 1)) ;
        while (want > 0 && (double)(f.mass_above + (want - 1) * w) >= goal) --want;
        while (want < f.in && (double)(f.mass_above + want * w) < goal) ++want;
      }
      limit_ties(r, value_of(kl), want);
      return false;
    }
    above = f.above;
    mass_above = f.mass_above;
    b = Bins(value_of(kl), value_of(kh));
  }
}

template <typename T, bool SMEM>
__global__ void __launch_bounds__(kNT, 2) sample_kernel(SampleArgs p) {
  extern __shared__ __align__(16) uint8_t smem[];
  using R = Row<T, SMEM>;
  constexpr int kVec = R::kVec;
  R r;
  Shared* s = r.s = reinterpret_cast<Shared*>(smem);
  float* vals = reinterpret_cast<float*>(smem + sizeof(Shared));
  r.vals = vals;
  r.ctas = p.ctas;
  r.arrive_started();
  r.rank = (int)(blockIdx.x % p.ctas);
  r.tid = threadIdx.x;
  r.lane = r.tid & 31;
  r.warp = r.tid >> 5;
  r.slice = p.slice;
  r.base = r.rank * p.slice;
  r.tau = -INFINITY;
  r.limit = 0;
  r.vec = p.vec;
  const int b = blockIdx.x / p.ctas;
  r.row = static_cast<const T*>(p.logits) + b * p.row_stride + r.base;
  r.n = max(0, min(p.slice, p.V - r.base));

  if (r.tid < 64) s->exp2_table[r.tid] = exp2((double)r.tid * (1.0 / 64));

  // ---- the slice's maximum (and the slice into shared memory), four vectors
  //      in flight a thread
  float most = -INFINITY;
  auto put = [&](int i, float v) {
    if constexpr (SMEM) vals[i] = v;
    most = fmaxf(most, v);  // not NaN
  };
  constexpr int kFly = 4;
  const int whole = p.vec ? r.n / kVec * kVec : 0;
  for (int i0 = r.tid * kVec; i0 < whole; i0 += kFly * kNT * kVec) {
    uint4 q[kFly];
#pragma unroll
    for (int f = 0; f < kFly; ++f) {
      const int i = i0 + f * kNT * kVec;
      if (i < whole) q[f] = *reinterpret_cast<const uint4*>(r.row + i);
    }
#pragma unroll
    for (int f = 0; f < kFly; ++f) {
      const int i = i0 + f * kNT * kVec;
      if (i >= whole) break;
#pragma unroll
      for (int j = 0; j < kVec; ++j) put(i + j, to_f32(reinterpret_cast<const T*>(&q[f])[j]));
    }
  }
  for (int i = whole + r.tid; i < r.n; i += kNT) put(i, to_f32(r.row[i]));
  if constexpr (SMEM)
    for (int i = r.n + r.tid; i < p.slice; i += kNT) vals[i] = -INFINITY;

  const double u = fmax((double)p.u[b], 0.0);  // NaN counts as 0
  float temp = p.temperature ? p.temperature[b] : p.temperature0;
  int k = p.top_k ? p.top_k[b] : p.top_k0;
  const double tp = p.top_p ? p.top_p[b] : p.top_p0;
  const double mp = fmax((double)(p.min_p ? p.min_p[b] : p.min_p0), 0.0);
  if (!(temp > 0.f)) k = 1;

  // Maximum of the row. And, for 1 to 512 sets of a CTA's threads: the least
  // maximum over the sets. As many logits as there are sets are at least that
  // large, which bounds the k-th largest from below.
  uint32_t set = key_of(most);
#pragma unroll
  for (int g = 5; g >= 0; --g) {  // sets of 32 >> g threads
    const uint32_t least = __reduce_min_sync(0xffffffffu, set);
    if (r.lane == 0) s->warp_u32[1 + g][r.warp] = least;
    if (g) set = max(set, __shfl_xor_sync(0xffffffffu, set, 32 >> g));
  }
  if (r.lane == 0) s->warp_u32[0][r.warp] = set;
  if (r.tid == 0) {
    s->first = INT32_MAX;
    s->n_list = 0;
  }
  __syncthreads();
  r.wait_started();
  if (r.warp >= 1 && r.warp <= 5) {  // sets of less than a warp
    const uint32_t x = __reduce_min_sync(0xffffffffu, r.lane < kWarps ? s->warp_u32[1 + r.warp][r.lane] : 0xffffffffu);
    if (r.lane < r.ctas) r.peer(r.lane)->peer_least[4 + r.warp][r.rank] = x;
  } else if (r.warp == 0) {  // of 1, 2, .. 16 warps: lanes 16 to 31 repeat the first
    uint32_t x = s->warp_u32[0][r.lane % kWarps];
#pragma unroll
    for (int g = 4; g >= 0; --g) {
      const uint32_t least = __reduce_min_sync(0xffffffffu, x);
      if (r.lane < r.ctas) r.peer(r.lane)->peer_least[g][r.rank] = least;
      if (g) x = max(x, __shfl_xor_sync(0xffffffffu, x, 16 >> g));
    }
    if (r.lane < r.ctas) r.peer(r.lane)->peer_max[r.rank] = x;
  }
  r.sync();
  uint32_t top = 0;
  for (int i = 0; i < r.ctas; ++i) top = max(top, s->peer_max[i]);
  if (top == 0) {
    if (r.rank == 0 && r.tid == 0) {
      p.token[b] = -1;
      p.logprob[b] = -INFINITY;
    }
    return;
  }
  r.top = value_of(top);
  r.flat = r.top == INFINITY;
  if (r.flat) {
    r.tau = r.top;
    r.limit = INT32_MAX;
  }
  r.c = 1.4426950408889634 / (double)temp;
  r.shift = p.shift;

  if (k == 1) {  // the lowest id of the largest logit
    int at = INT32_MAX;
    r.each([&](const float (&l)[4], int i) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (l[j] == r.top) at = min(at, i + j + r.base);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (r.lane == 0 && at != INT32_MAX) atomicMin(&r.peer(0)->first, at);
    r.sync();
    if (r.rank == 0 && r.tid == 0) {
      p.token[b] = s->first;
      p.logprob[b] = 0.f;
    }
    return;
  }
  if (k > 0 && k < p.V) {
    int g = 0;  // the largest sets that are at least k
    while (g < kGroups && (r.ctas << g) < k) ++g;
    uint32_t least = 0;
    if (g < kGroups) {
      least = 0xffffffffu;
      for (int i = 0; i < r.ctas; ++i) least = min(least, s->peer_least[g][i]);
    }
    const float lo = least ? value_of(least) : -FLT_MAX;  // 0: an empty set among them
    // About g ln g of the logits reach the least of g maxima, whatever their
    // distribution: few enough for the list without a histogram.
    if (least && (r.ctas << g) <= 128) {
      gather(r, [&](float l) { return l >= lo; });
      const uint32_t found = r.peer(0)->n_list;
      r.sync();  // read before the first CTA goes on
      if (found <= kCap) {
        if (r.rank == 0) finish_list(r, (int)found, k, tp, mp, u, 0, p.token + b, p.logprob + b);
        return;
      }
    }
    if (select<false>(r, lo, (double)k, k, tp, mp, u, p.token + b, p.logprob + b)) return;
  }
  if (tp < 1.0) {
    // tokens of weight below (1 - p) / 2V hold less than 1 - p of the mass, as
    // the largest alone weighs 1: the boundary lies above them
    const double eps = (1.0 - tp) / (2.0 * (double)p.V);
    const float bound = r.flat ? r.top : (float)(r.top + log2(eps) / r.c * 1.0001 - fabs((double)r.top) * 3e-7);
    const float lo = bound > -FLT_MAX ? fminf(bound, r.top) : -FLT_MAX;
    if (select<true>(r, lo, 0.0, k, tp, mp, u, p.token + b, p.logprob + b)) return;
  }

  // ---- draw from the whole row: masses of contiguous blocks, one per warp
  const int per = p.slice / kWarps, i0 = r.warp * per;
  // logits this low have w < mp for certain, as w is computed: 1e-9 of the
  // exponent covers its error, at temperatures where every weight rounds to 1 too
  const float low = mp > 0.0 && !r.flat
                        ? (float)(r.top + (log2(mp) - 1e-9) / r.c * 1.0001 - fabs((double)r.top) * 3e-7) : -INFINITY;
  auto may = [&](float l, int i) { return (l >= low || l == r.top) && r.kept(l, r.base + i); };
  auto share = [&](float l, double w) { return w >= mp || l == r.top ? r.units(w) : 0; };
  u64 sum = 0;
  r.each(i0, i0 + per, r.lane, 32, [&](const float (&l)[4], int i) {
    bool in[4], any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) any |= in[j] = may(l[j], i + j);
    if (!any) return;
    double w[4];
    r.weights(l, w);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (in[j]) sum += share(l[j], w[j]);
  });
  sum = r.warp_add(sum);
  __syncthreads();
  if (r.lane == 0) s->warp_sum[r.warp] = sum;
  if (r.tid == 0) s->owner = -1;
  __syncthreads();
  if (r.tid < r.ctas) {
    u64 t = 0;
    for (int i = 0; i < kWarps; ++i) t += s->warp_sum[i];
    r.peer(r.tid)->peer_mass[r.rank] = t;
  }
  r.sync();
  u64 z = 0, before = 0;
  for (int i = 0; i < r.ctas; ++i) {
    if (i < r.rank) before += s->peer_mass[i];
    z += s->peer_mass[i];
  }
  for (int i = 0; i < r.warp; ++i) before += s->warp_sum[i];
  double goal = u * (double)z;
  if (!(goal < (double)z)) goal = below((double)z);
  // the one block in which the running mass passes the goal is split again
  // over the warps of its CTA
  auto holds = [&](u64 from, u64 mass) { return mass && !((double)from > goal) && (double)(from + mass) > goal; };
  if (holds(before, sum) && r.lane == 0) {
    s->owner = r.warp;
    s->peer_total[0] = before;
  }
  __syncthreads();
  if (s->owner < 0) return;
  const int part = (per / kWarps + 31) / 32 * 32, j0 = s->owner * per, j1 = j0 + per;
  const int p0 = min(j0 + r.warp * part, j1), p1 = min(p0 + part, j1);
  before = s->peer_total[0];
  sum = 0;
  for (int i = p0 + r.lane; i < p1; i += 32) {
    const float l = r.at(i);
    if (may(l, i)) sum += share(l, r.weight(l));
  }
  sum = r.warp_add(sum);
  __syncthreads();
  if (r.lane == 0) s->warp_sum[r.warp] = sum;
  __syncthreads();
  for (int i = 0; i < r.warp; ++i) before += s->warp_sum[i];
  if (!holds(before, sum)) return;
  for (int i = p0; i < p1; i += 32) {
    const float l = r.at(i + r.lane);  // blocks are whole warps wide
    const double w = r.weight(l);
    const u64 own = may(l, i + r.lane) ? share(l, w) : 0;
    u64 x = own;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const u64 up = __shfl_up_sync(0xffffffffu, x, off);
      if (r.lane >= off) x += up;
    }
    const uint32_t any = __ballot_sync(0xffffffffu, own && (double)(before + x) > goal);
    if (any) {
      if (r.lane == __ffs(any) - 1) {
        p.token[b] = r.base + i + r.lane;
        p.logprob[b] = (float)log(w / r.weight_of(z));
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, x, 31);
  }
}

template <typename T, bool SMEM>
int launch_on(const SampleArgs& a, int B, cudaStream_t st) {
  const int bytes = (int)sizeof(Shared) + (SMEM ? a.slice * 4 : 0);
  // The limit belongs to the function and every host thread shares it, so it is
  // the same constant whatever the call: a smaller one would refuse another
  // thread's launch.
  constexpr int most = (int)sizeof(Shared) + kSmemSlice * 4;
  if (SMEM)
    WKVM_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T, SMEM>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  if (a.ctas > 8)
    WKVM_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T, SMEM>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)B * a.ctas));
  cfg.blockDim = dim3(kNT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, SMEM>, a) == cudaSuccess ? WKVM_OK : WKVM_ERR_CUDA;
}

template <typename T>
int launch(const SampleArgs& a, int B, cudaStream_t st) {
  return a.slice <= kSmemSlice ? launch_on<T, true>(a, B, st) : launch_on<T, false>(a, B, st);
}

}  // namespace
}  // namespace wkvm

extern "C" int wkvm_sample_tokens(const void* logits, int64_t row_stride, const float* u,
                                  const float* temperature, const int32_t* top_k,
                                  const float* top_p, const float* min_p, float temperature0,
                                  int32_t top_k0, float top_p0, float min_p0, int64_t* tokens,
                                  float* logprobs, int32_t B, int32_t V, int32_t dtype,
                                  int32_t* status, wkvm_stream_t stream) {
  (void)status;  // nothing in a row can be wrong on the device
  if (B < 0 || V <= 0) return WKVM_ERR_INVALID_ARG;
  if (dtype != WKVM_DTYPE_F32 && dtype != WKVM_DTYPE_BF16 && dtype != WKVM_DTYPE_F16)
    return WKVM_ERR_DTYPE;
  if (V > WKVM_SAMPLE_MAX_VOCAB) return WKVM_ERR_SHAPE;
  if (B == 0) return WKVM_OK;
  if (!logits || !u || !tokens || !logprobs) return WKVM_ERR_INVALID_ARG;
  // Slices of 16,384 fit shared memory and spread the rows that need several
  // passes among those that do not: 256 rows of 65,536 with a mix of settings
  // take 90 us over four CTAs each, 99 over two, 140 whole, 106 over eight. Rows
  // that all need them gain nothing and pay the barriers: top-p for all 170 us
  // over four, 158 over two, 154 whole; greedy 25, 24 and 20. Few rows take more
  // CTAs (one under top-p: 21 us over sixteen, 24 over eight, 33 over four, 88
  // whole; 32 mixed rows 33 over eight, 37 over sixteen), sixteen only where all
  // are resident at once.
  int ctas = 1;
  while (ctas < 8 && (V > ctas * wkvm::kSmemSlice || ((int64_t)B * ctas <= 256 && V >= ctas * 2048))) ctas *= 2;
  if (ctas == 8 && (B <= 8 || V > 8 * wkvm::kSmemSlice) && V >= 16384) ctas = 16;
  if ((int64_t)B * ctas > INT32_MAX) return WKVM_ERR_SHAPE;
  const int64_t es = dtype == WKVM_DTYPE_F32 ? 4 : 2;
  const int slice = ((V + ctas - 1) / ctas + wkvm::kNT - 1) / wkvm::kNT * wkvm::kNT;
  const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (B == 1 || row_stride * es % 16 == 0);
  double shift = 1.0;  // s = min(52, 62 - ceil(log2 V))
  for (int64_t v = 1 << 10; v < V; v *= 2) shift *= 2.0;
  wkvm::SampleArgs a{logits, row_stride, u, temperature, top_p, min_p, top_k, temperature0, top_p0,
                     min_p0, top_k0, tokens, logprobs, V, slice, ctas, shift, vec};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case WKVM_DTYPE_F32: return wkvm::launch<float>(a, B, st);
    case WKVM_DTYPE_BF16: return wkvm::launch<__nv_bfloat16>(a, B, st);
    default: return wkvm::launch<__half>(a, B, st);
  }
}
