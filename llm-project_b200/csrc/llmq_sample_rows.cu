// llmq_sample_rows.cu - one token for each row of a batch of logits, by
// temperature, top-k, min-p and top-p, from given random numbers
// (llmq_sample_rows).
//
// A row's weights are w_j = exp((l_j - max l) / T), as 64-bit integers: w_j is
// rounded to a whole number of 2^-S, S = min(50, 62 - ceil(log2 vocab)), so any
// sum of them is exact, fits 63 bits and is the same in any order.  The tokens'
// order is ord = (the logit's bits mapped to an unsigned key of the same order) *
// 2^20 + 2^20 - 1 - index, larger first (key 0: NaN and -infinity, never drawn).
// Each of the three cuts keeps a prefix of that order, so what is kept is known
// by its sum alone, and the draw is the first token at which the sum reaches u
// times the kept one.  No cut needs a sorted row: only the tokens around it.
//
// A cluster of CTAs shares a row, which is read from DRAM once: each CTA keeps its slice in
// shared memory if that has room (64 KB: 8 CTAs for 128256 f32 logits, 4 for f16), else
// later passes read it from L2.
//  1. The largest and least logit, and for a top_k up to 96 the largest of each of
//     128 groups of tokens: the k-th largest of those is a bound that at least k
//     tokens reach and few more do (k = 40: about 48 of a smooth row's).  A min_p
//     gives another bound.
//  2. With a bound, the tokens that reach it go to the first CTA's list (the whole
//     sum, where top_p asks for it, is formed on the way).  The list is sorted and
//     everything follows from its prefix sums.
//  3. Without one (or if the list overflows), a histogram of exact sums (and counts,
//     for a top_k) over kBins steps of the logit.  A prefix sum finds the step each
//     cut lies in, which bounds the kept sum and so the steps the draw can be in; the
//     tokens of these few steps are listed and sorted.  If they are too many (rows of
//     ties), the cuts and the draw go one by one, dividing a step by ord, down to
//     single tokens if need be.
//
// What bounds it is not DRAM but instructions and latency: a weight costs some 30
// instructions (doubles, for the exact sum), the histogram two shared atomics a token.
// Measured: 64 f32 rows of 128256 with mixed settings (32.8 MB, 5.1 us at a plain copy's
// rate) 56 to 59 us, the time of their rows without a bound, which share 4 CTAs like all
// others (64 of those alone: 58; 256: 161; f16: 57 and 151); the same rows with a top_k of 50,
// no exponential but the list's, 24 us, and with a top_k of 40 and a top_p, which asks for the
// whole sum, 37.5; one row of 32000 so 10.5 us, a chain of cluster barriers.  Counters for
// the mixed rows: 33.0 MB read, 40% of the issue slots, two further turns of a shared
// atomic for equal banks.
#include <cfloat>
#include <climits>
#include <cmath>
#include <cooperative_groups.h>
#include <type_traits>

#include "llmq_serve.cuh"

using namespace llmq;
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;
constexpr int kThreads = 512;
constexpr int kBins = 1024;
constexpr int kListCap = 2048;
constexpr int kMaxCluster = 8;
constexpr int kGroups = 128;  // groups of tokens whose maxima bound a top_k
constexpr int kIndexBits = 20;

__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __float_as_uint(__fadd_rn(l, 0.0f));  // -0 to +0: equal logits, equal keys
  if (!(l > -INFINITY)) return 0u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // order_key's value for it but for the exclusion
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 token_ord(uint32_t key, int j) {
  return (static_cast<u64>(key) << kIndexBits) | static_cast<u64>((1 << kIndexBits) - 1 - j);
}

// exp on the way to an integer: 2^(-y / 256) for y = (max - l) * 256 log2(e) / T as
// 2^-(n / 256), n the integer next to y, from a table of 2^-(i / 256), times the
// Taylor polynomial of 2^(-x / 256), |x| = |y - n| <= 1/2, up to x^4 (the rest: 2^-54).
constexpr int kExpTable = 256;
struct RowRule {
  float mx;            // the largest logit
  bool infinite;       // it is +infinity: only its equals count, whatever T
  double mxd, step;    // step: 256 log2(e) / T
  int scale;           // S
  const double *tab;   // shared: 2^(S - i / 256)
  float bin_scale;     // steps of the histogram a unit of logit

  uint32_t far;        // high word of 256 (S + 1): a y from there on has a w that rounds to 0

  // w * 2^S before rounding, as a product; counts: it does not round to 0 (false for NaN
  // and -infinity; the product is then nothing).
  //
  // A token's weight is formed at several places (histogram, whole sum, list, divided step),
  // whose sums have to agree to the unit.  So each operation names its rounding: left to
  // the compiler, which may make one operation of a product and a sum at one place and
  // two at another, one weight in 70 could differ by a unit.
  struct Product {
    double p, t;
    bool counts;
  };
  static constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: the integer in the low bits
  __device__ __forceinline__ Product product(float l) const {  // not for an infinite maximum
    const double y = __dmul_rn(__dsub_rn(mxd, static_cast<double>(l)), step);  // >= 0, or NaN
    const double yr = __dadd_rn(y, kRound);
    const int n = __double2loint(yr);
    const double x = __dsub_rn(y, __dsub_rn(yr, kRound));
    constexpr double c = -2.7076061740622863e-3;  // -ln 2 / 256
    double p = __fma_rn(x, c * c * c * c / 24.0, c * c * c / 6.0);
    p = __fma_rn(x, p, c * c / 2.0);
    p = __fma_rn(x, p, c);
    p = __fma_rn(x, p, 1.0);
    const double t = tab[n & (kExpTable - 1)];  // of 2^S 2^(-i / 256)
    const bool counts = static_cast<uint32_t>(__double2hiint(y)) < far;  // as unsigned: no NaN of either sign
    return Product{p, __hiloint2double(__double2hiint(t) - ((n >> 8) << 20), __double2loint(t)), counts};
  }
  // the product next to an integer, rounded once (it is below 2^51)
  static __device__ __forceinline__ u64 rounded(const Product &e) {
    return static_cast<u64>(__double_as_longlong(__fma_rn(e.p, e.t, kRound))) - 0x4338000000000000ull;
  }
  __device__ __forceinline__ Product product_any(float l) const {
    if (infinite) return Product{1.0, __hiloint2double((1023 + scale) << 20, 0), l == mx};
    return product(l);
  }
  __device__ __forceinline__ double share(const Product &e) const { return e.counts ? __dmul_rn(e.p, e.t) : 0.0; }
  __device__ __forceinline__ u64 weight(const Product &e) const { return e.counts ? rounded(e) : 0ull; }
  __device__ __forceinline__ double share(float l) const { return share(product_any(l)); }
  __device__ __forceinline__ u64 weight(float l) const { return weight(product_any(l)); }
  // the histogram's step: any function that does not fall as l falls will do (the
  // integer next to the product; NaN goes last)
  __device__ __forceinline__ int bin(float l) const {
    const float x = fminf((mx - l) * bin_scale, static_cast<float>(kBins - 1)) + 8388608.0f;
    return __float_as_int(x) & (kBins - 1);
  }
  __device__ __forceinline__ void set(float high, float temp, int bits, const double *table) {
    mx = __fadd_rn(high, 0.0f);  // +0, not -0: no difference below is -0
    infinite = high == INFINITY;
    mxd = static_cast<double>(mx);
    step = kExpTable * 1.4426950408889634 / static_cast<double>(temp);
    scale = bits;
    far = static_cast<uint32_t>(__double2hiint(kExpTable * static_cast<double>(bits + 1)));
    tab = table;
    bin_scale = 0.0f;
  }
};

struct Command {
  int op;           // what the cluster does next
  int bin0, bin1;   // tokens of these steps
  u64 lo, hi;       // and of this range of ord
  int shift;        // op kDivide: the new step is (hi - ord) >> shift
};
enum { kDone = 0, kGather = 1, kDivide = 2 };

// A step of the histogram: its sum and tokens, and those before it.
struct Step {
  int bin, before_n, count;
  u64 before, mass;
};

// What each CTA keeps in static shared memory; the first CTA's is the row's.
struct Shared {
  double tab[kExpTable];
  u64 red[kThreads / 32];
  u64 whole[kMaxCluster], above[kMaxCluster];
  float high[kMaxCluster], low[kMaxCluster], warp_high[kThreads / 32], warp_low[kThreads / 32];
  int listed;        // tokens gathered here
  int total;         // the row's list (first CTA)
  int place;         // where this CTA's part of it goes
  __align__(16) uint32_t groups[kGroups];
  uint32_t pick_key;
  int pick_bin, pick_count;
  u64 pick_before, pick_before_count;
  int pick_item;     // of a greedy row
  int found[2];      // a list's item, -1: none (the calls take the places in turn)
  u64 found_sum[2];
  int last;          // the list's last item of a weight, and its sum
  u64 last_sum;
  u64 sum, tokens;
  Step step[4];  // the top_p cut's, the top_k's, the least and the most the draw can be in
  Command cmd;
};

__device__ __forceinline__ u64 warp_scan(u64 v) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}
// Inclusive sum over the block's threads (*all: of all of them); every thread of the
// block calls this.
template <int NT = kThreads>
__device__ __forceinline__ u64 block_scan(u64 v, u64 *red, u64 *all = nullptr) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan(v);
  __syncthreads();
  if (lane == 31) red[warp] = v;
  __syncthreads();
  const u64 w = warp_scan(lane < NT / 32 ? red[lane] : 0);
  const u64 before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  if (all) *all = __shfl_sync(0xffffffffu, w, 31);
  return warp ? v + before : v;
}
__device__ __forceinline__ u64 block_sum(u64 v, u64 *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
  for (int o = kThreads / 64; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ceil(f * total) in 1 .. total
__device__ __forceinline__ u64 part_of(double f, u64 total) {
  const double t = ceil(f * static_cast<double>(total));
  const u64 v = t < 1.0 ? 1ull : static_cast<u64>(t);
  return v > total ? total : v;
}

// Dynamic shared memory: the histogram (counts, then the sums' low and high
// words) or this CTA's gathered tokens; the row's histogram; the row's list or
// the histogram of a divided step; the slice of the row.
constexpr int kHistBytes = kBins * 12;
constexpr int kListBytes = kListCap * 8;
constexpr int kWorkBytes = kListBytes + kHistBytes + kListBytes;
static_assert(kHistBytes <= kListBytes, "regions are shared");

constexpr int kMaxResident = 64 * 1024;  // of the slice

struct RowArgs {
  LlmqSampleRows a;
  int slice;     // tokens a CTA, a multiple of 16
  int resident;  // the slice is kept in shared memory
  int scale;     // S
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample_rows(const RowArgs p) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  __shared__ Shared sh;
  constexpr int kVec = 16 / sizeof(T);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  uint32_t *bin_count = reinterpret_cast<uint32_t *>(s_dyn), *bin_lo = bin_count + kBins;
  u64 *gathered = reinterpret_cast<u64 *>(s_dyn);
  u64 *tot_mass = reinterpret_cast<u64 *>(s_dyn + kListBytes);
  uint32_t *tot_count = reinterpret_cast<uint32_t *>(tot_mass + kBins);
  u64 *list = reinterpret_cast<u64 *>(s_dyn + kListBytes + kHistBytes);
  T *slice = reinterpret_cast<T *>(s_dyn + kWorkBytes);
  Shared *first = cluster.map_shared_rank(&sh, 0);

  const LlmqSampleRows &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / ctas, j0 = rank * p.slice, n = max(0, min(p.slice, a.vocab - j0));
  cluster.barrier_arrive();  // every CTA runs before any writes to another
  if (tid < kExpTable) sh.tab[tid] = exp2(p.scale - tid * (1.0 / kExpTable));
  if (tid == 0) {
    sh.listed = sh.total = 0;
    sh.pick_item = INT_MAX;
    sh.found[0] = sh.found[1] = -1;
    sh.last = 0;
    sh.last_sum = 0;
  }
  serve_wait();
  serve_dependents();
  const T *row = static_cast<const T *>(a.logits) + r * a.stride + j0;
  const float temp = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  const float min_p = a.min_p && a.min_p[r] > 0.0f ? fminf(a.min_p[r], 1.0f) : 0.0f;
  const float top_p = a.top_p && a.top_p[r] > 0.0f && a.top_p[r] < 1.0f ? a.top_p[r] : 0.0f;
  const int top_k = a.top_k && a.top_k[r] > 0 && a.top_k[r] < a.vocab ? a.top_k[r] : 0;

  // f(kVec logits, index of the first) over the slice, the next vector on its way
  // meanwhile; the ends that fill no vector come one by one, with NaN beside them
  const T *src = p.resident ? slice : row;
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / sizeof(T)));
  const int nv = (n - head) / kVec;
  auto each = [&](auto f) {
    const Pack<T, kVec> *vec = reinterpret_cast<const Pack<T, kVec> *>(src + head);
    Pack<T, kVec> next;
    if (tid < nv) next = vec[tid];
    float l[kVec];
    for (int v = tid; v < nv; v += kThreads) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) l[i] = to_f32(next.v[i]);
      if (v + kThreads < nv) next = vec[v + kThreads];
      f(l, j0 + head + v * kVec);
    }
    const int e = tid < head ? tid : tid + kVec * nv;  // fewer than 2 kVec of them
    if (tid < n - kVec * nv) {
#pragma unroll
      for (int i = 1; i < kVec; ++i) l[i] = NAN;
      l[0] = to_f32(src[e]);
      f(l, j0 + e);
    }
  };

  // ---- 1. the slice, its largest (with its first index) and least logit
  if (p.resident) {
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
#pragma unroll 4
      for (int v = tid; v < n / kVec; v += kThreads)
        reinterpret_cast<Pack<T, kVec> *>(slice)[v] = reinterpret_cast<const Pack<T, kVec> *>(row)[v];
      for (int j = n / kVec * kVec + tid; j < n; j += kThreads) slice[j] = row[j];
    } else {
#pragma unroll 4
      for (int j = tid; j < n; j += kThreads) slice[j] = row[j];
    }
    __syncthreads();
  }
  float high = -INFINITY, low = INFINITY;  // fmaxf and fminf pass over NaN
  each([&](const float *l, int) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      high = fmaxf(high, l[i]);
      low = fminf(low, l[i]);
    }
  });
  const float thread_high = high;
  {
    const int lanes = ctas * kThreads / kGroups;  // of a group: 4 .. 32
    float g = high;
    for (int o = 1; o < lanes; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    float hi = high, lo = low;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (lane == 0) {
      sh.warp_high[warp] = hi;
      sh.warp_low[warp] = lo;
    }
    __syncthreads();
    cluster.barrier_wait();
    if (top_k && tid % lanes == 0)
      for (int c = 0; c < ctas; ++c)
        cluster.map_shared_rank(&sh, c)->groups[(rank * kThreads + tid) / lanes] = order_key(g);
    if (tid < ctas) {
      for (int w = 0; w < kThreads / 32; ++w) {
        hi = fmaxf(hi, sh.warp_high[w]);
        lo = fminf(lo, sh.warp_low[w]);
      }
      Shared *to = cluster.map_shared_rank(&sh, tid);
      to->high[rank] = hi;
      to->low[rank] = lo;
    }
  }
  cluster.sync();
  for (int c = 0; c < ctas; ++c) {
    high = fmaxf(high, sh.high[c]);
    low = fminf(low, sh.low[c]);
  }
  if (high == -INFINITY) {  // nothing can be drawn
    if (rank == 0 && tid == 0) {
      a.ids[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  if (greedy) {  // the first of the largest
    int at = INT_MAX;
    each([&](const float *l, int j) {
#pragma unroll
      for (int i = kVec - 1; i >= 0; --i)
        if (l[i] == high) at = min(at, j + i);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0 && at != INT_MAX) atomicMin(&first->pick_item, at);
    cluster.sync();
    if (rank == 0 && tid == 0) {
      a.ids[r] = sh.pick_item;
      if (a.logprobs) a.logprobs[r] = 0.0f;
    }
    return;
  }
  const u64 top = token_ord(order_key(high), 0);  // no token's ord is larger
  RowRule rule;
  rule.set(high, temp, p.scale, sh.tab);
  {
    // steps over what the row spans, or down to weights that round to nothing
    const float span = fminf(high - low, 36.0f * temp);
    if (span > 0.0f && span < INFINITY) rule.bin_scale = fminf(kBins / span, 1e30f);
  }

  // ---- a bound that the tokens of every cut reach
  uint32_t bound = 0;
  bool bounded = a.vocab <= kListCap;
  if (!bounded && top_k && top_k <= kGroups * 3 / 4) {
    // the top_k-th largest of the groups' maxima: four threads count what precedes each
    constexpr int kParts = kThreads / kGroups;
    const int g = tid / kParts, part = tid % kParts;
    const uint32_t mine = sh.groups[g];
    int before = 0;
#pragma unroll
    for (int i = 0; i < kGroups / kParts; ++i) {
      const int x = part + kParts * i;
      const uint32_t k = sh.groups[x];
      before += k > mine || (k == mine && x < g);
    }
    for (int o = 1; o < kParts; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (before == top_k - 1) sh.pick_key = mine;
    __syncthreads();
    bound = sh.pick_key;
    bounded = true;
  }
  if (min_p > 0.0f) {
    // l >= max + T ln(min_p), a little lower: the list is cut exactly
    const double at = rule.mxd + static_cast<double>(temp) * log(static_cast<double>(min_p)) * (1.0 + 1e-6);
    const uint32_t k = order_key(__double2float_rd(at - 1e-6 * fabs(rule.mxd)));
    bound = max(bound, min(k, order_key(high)));
    bounded = true;
  }

  // ---- 2. the tokens that reach the bound
  // Lists what is wanted of the logits in [lo, hi] (a first, cheap look), at most a few
  // thousand tokens of a row, one atomic each: into `gathered`, then to the first
  // CTA's list.
  auto gather = [&](float lo, float hi, auto wanted) {
    each([&](const float *l, int j) {
      uint32_t want = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) want |= l[i] >= lo && l[i] <= hi ? 1u << i : 0u;
      if (want) {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (((want >> i) & 1u) && wanted(l[i], j + i)) {
            const int at = atomicAdd(&sh.listed, 1);
            if (at < kListCap) gathered[at] = token_ord(order_key(l[i]), j + i);
          }
      }
    });
    __syncthreads();
    const int mine = sh.listed;
    if (tid == 0) sh.place = mine ? atomicAdd(&first->total, mine) : 0;
    __syncthreads();
    u64 *to = cluster.map_shared_rank(list, 0);
    for (int i = tid; i < min(mine, kListCap); i += kThreads)
      if (sh.place + i < kListCap) to[sh.place + i] = gathered[i];
    if (tid == 0) sh.listed = 0;
  };
  // logits that all tokens of steps b0 .. b1 lie between
  const float width = rule.bin_scale > 0.0f ? 1.0f / rule.bin_scale : INFINITY;
  auto over_step = [&](int b) { return b > 0 && width < INFINITY ? high - width * static_cast<float>(b - 1) : INFINITY; };
  auto under_step = [&](int b) {
    return b < kBins - 1 && width < INFINITY ? fmaxf(high - width * static_cast<float>(b + 1), -FLT_MAX) : -FLT_MAX;
  };
  const double min_share = static_cast<double>(min_p) * static_cast<double>(1ull << p.scale);
  u64 whole = 0, above = 0;
  if (bounded) {
    const float least = bound > kKeyNegInf ? key_logit(bound) : -FLT_MAX;
    // A min_p says nothing of how many tokens reach it.  Of kThreads threads with a share
    // of the slice each, `over` have one that does: some -kThreads ln(1 - over / kThreads)
    // tokens.  Half again too many for the list: it overflows without being tried.
    const int over = __syncthreads_count(thread_high >= least);
    const bool hopeless = a.vocab > kListCap &&
                          -kThreads * logf(1.0f - over / (kThreads + 0.5f)) > 1.5f * kListCap / ctas;
    if (hopeless && tid == 0) atomicAdd(&first->total, kListCap + 1);
    if (!hopeless) gather(least, INFINITY, [](float, int) { return true; });
    if (top_p > 0.0f && !hopeless) each([&](const float *l, int) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) whole += rule.weight(l[i]);
      });
  } else {
    for (int b = tid; b < 3 * kBins; b += kThreads) bin_count[b] = 0;
    __syncthreads();
  }
  // Adds N weights to their steps, those that count: the low words first, all on their
  // way at once, then the high words with what the low ones carried.
  const uint32_t lo_addr = static_cast<uint32_t>(__cvta_generic_to_shared(bin_lo));
  auto count_in = [&](const auto &w, const auto &b, const auto &counts, auto counted) {
    constexpr int N = sizeof(w) / sizeof(w[0]);
    uint32_t old[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      asm volatile(
          "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %3, 0;\n\t@q atom.shared.add.u32 %0, [%1], %2;\n\t}"
          : "=&r"(old[i])
          : "r"(lo_addr + 4 * b[i]), "r"(static_cast<uint32_t>(w[i])), "r"(counts[i] ? 1u : 0u)
          : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t lo = static_cast<uint32_t>(w[i]), hi = static_cast<uint32_t>(w[i] >> 32) + (old[i] + lo < old[i] ? 1u : 0u);
      asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q red.shared.add.u32 [%0+%3], %1;\n\t}" ::"r"(
                       lo_addr + 4 * b[i]),
                   "r"(hi), "r"(counts[i] ? hi : 0u), "n"(4 * kBins)
                   : "memory");
      if (counted.value && counts[i]) atomicAdd(&bin_count[b[i]], 1u);
    }
  };
  // `all`: with counts (of a top_k) and the sum of w >= min_p, for any maximum
  auto fill = [&](auto all) {
    each([&](const float *l, int) {
#pragma unroll
      for (int h = 0; h < kVec; h += 4) {
        u64 w[4];
        int b[4];
        bool counts[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (all.value) {
            const RowRule::Product e = rule.product_any(l[h + i]);
            w[i] = rule.weight(e);
            counts[i] = w[i] != 0;
            above += rule.share(e) >= min_share ? w[i] : 0;
          } else {
            const RowRule::Product e = rule.product(l[h + i]);
            w[i] = RowRule::rounded(e);
            counts[i] = e.counts;
          }
          b[i] = rule.bin(l[h + i]);
        }
        count_in(w, b, counts, all);
      }
    });
  };
  auto histogram = [&]() {
    if (top_k || min_p > 0.0f || rule.infinite)
      fill(std::true_type());
    else
      fill(std::false_type());
  };
  // the row's histogram, each CTA summing a part of the steps: in every CTA, or (of a
  // divided step) in the first
  auto collect = [&](u64 *mass, uint32_t *count, int receivers) {
    cluster.sync();
    const int each_bins = kBins / ctas;
    for (int i = tid; i < each_bins; i += kThreads) {
      const int b = rank * each_bins + i;
      u64 m = 0;
      uint32_t cnt = 0;
      for (int c = 0; c < ctas; ++c) {
        const uint32_t *h = cluster.map_shared_rank(bin_count, c);
        m += h[kBins + b] + (static_cast<u64>(h[2 * kBins + b]) << 32);
        if (top_k) cnt += h[b];
      }
      for (int c = 0; c < receivers; ++c) {
        cluster.map_shared_rank(mass, c)[b] = m;
        cluster.map_shared_rank(count, c)[b] = cnt;
      }
    }
  };
  auto publish = [&](u64 v, u64 (Shared::*to)[kMaxCluster]) {
    v = block_sum(v, sh.red);
    if (tid < ctas) (cluster.map_shared_rank(&sh, tid)->*to)[rank] = v;
  };
  bool have_hist = !bounded;
  if (bounded) {
    if (top_p > 0.0f) publish(whole, &Shared::whole);
    cluster.sync();
    have_hist = first->total > kListCap;  // too many reach the bound: by the histogram after all
    cluster.barrier_arrive();             // the first CTA outlives the others' look at its memory
    if (!have_hist && rank != 0) return;
    if (have_hist) {
      cluster.barrier_wait();
      if (rank == 0 && tid == 0) sh.total = 0;  // the next listing comes after the histogram's barriers
      for (int b = tid; b < 3 * kBins; b += kThreads) bin_count[b] = 0;
      __syncthreads();
    }
  }
  if (have_hist) {
    histogram();
    if (min_p > 0.0f) publish(above, &Shared::above);
    collect(tot_mass, tot_count, ctas);
    cluster.sync();
  }

  // sorts list[0 .. m) by falling ord, m <= kListCap (bitonic).  A warp's pairs of a
  // stride up to 32 stay within its 64 items: only larger strides need the other warps,
  // and a list of up to 64 items one warp alone.
  // Up to kCounted items are put in place by counting what precedes each, several
  // threads an item; the sorted items are then in `gathered`.  (64 f32 rows of 128256 with a
  // top_k of 50, whose lists hold some 60: 24.2 us, 26.7 sorted; nucleus rows, of a few
  // hundred: 60.7 us counted up to 512, 58.0 up to 256.)
  constexpr int kCounted = 256;
  static_assert(kCounted <= kThreads, "a thread an item");
  u64 *items = list;
  auto sort_list = [&](int m) {
    if (m <= kCounted) {
      int parts = 1;  // threads an item, 32 at most
      while (parts < 32 && m * parts * 2 <= kThreads) parts *= 2;
      const int x = tid / parts;
      int before = 0;
      if (x < m) {
        const u64 mine = list[x];
#pragma unroll 4
        for (int y = tid % parts; y < m; y += parts) before += list[y] > mine;
      }
      for (int o = 1; o < parts; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
      items = gathered;
      if (x < m && tid % parts == 0) items[before] = list[x];
      __syncthreads();
      return;
    }
    items = list;
    int size2 = 2;
    while (size2 < m) size2 <<= 1;
    for (int i = m + tid; i < size2; i += kThreads) list[i] = 0;
    __syncthreads();
    const int warps = max(1, min(kThreads, size2 / 2) / 32);
    if (warp < warps) {
      for (int size = 2; size <= size2; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
          for (int i = tid; i < size2 / 2; i += 32 * warps) {
            const int x = 2 * i - (i & (stride - 1)), y = x + stride;
            const u64 u = list[x], v = list[y];
            if ((u < v) == ((x & size) == 0)) {
              list[x] = v;
              list[y] = u;
            }
          }
          if (warps > 1 && (stride > 32 || (stride == 1 && size > 32)))
            asm volatile("bar.sync 1, %0;" ::"r"(32 * warps) : "memory");
          else
            __syncwarp();
        }
    }
    __syncthreads();
  };
  constexpr int kPer = kListCap / kThreads;
  // a sorted list's weights and sums: thread's items tid * kPer + i, sum up to and with each
  int m = 0;
  u64 w[kPer], sums[kPer];
  auto list_sums = [&](u64 before) {
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int x = tid * kPer + i;
      w[i] = x < m ? rule.weight(key_logit(static_cast<uint32_t>(items[x] >> kIndexBits))) : 0;
      mine += w[i];
    }
    u64 all;  // of the list
    u64 at = before + block_scan(mine, sh.red, &all) - mine;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      at += w[i];
      sums[i] = at;
      if (w[i] && at == before + all) {
        sh.last = tid * kPer + i;
        sh.last_sum = at;
      }
    }
  };
  // One thread's item, known to it, and its sum to all; if no thread has it (which sums
  // that agree rule out), the last item of a weight: always one of the list.
  int calls = 0;
  auto share_item = [&](auto is_it, u64 *sum_there) -> int {
    const int mine = calls & 1;
    ++calls;
    __syncthreads();
    if (tid == 0) sh.found[mine ^ 1] = -1;  // for the next call: the last one's is read
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (is_it(i)) {
        sh.found[mine] = tid * kPer + i;
        sh.found_sum[mine] = sums[i];
      }
    __syncthreads();
    const int item = sh.found[mine];
    *sum_there = item < 0 ? sh.last_sum : sh.found_sum[mine];
    return item < 0 ? sh.last : item;
  };
  // the first of the list's items whose sum reaches target (there is one), and its sum
  auto reach = [&](u64 target, u64 *sum_there) {
    return share_item([&](int i) { return w[i] && sums[i] >= target && sums[i] - w[i] < target; }, sum_there);
  };
  auto answer = [&](int item, u64 kept) {
    if (tid == 0) {
      const u64 o = items[item];
      const float l = key_logit(static_cast<uint32_t>(o >> kIndexBits));
      a.ids[r] = (1 << kIndexBits) - 1 - static_cast<int>(o & ((1 << kIndexBits) - 1));
      if (a.logprobs) {
        const double lw = l == rule.mx ? 0.0 : -(rule.mxd - static_cast<double>(l)) / static_cast<double>(temp);
        a.logprobs[r] = static_cast<float>(lw - log(ldexp(static_cast<double>(kept), -p.scale)));
      }
    }
  };
  const float uf = a.u[r];
  const double u = uf > 0.0f ? fminf(uf, 1.0f) : 0.0f;

  if (!have_hist) {  // the list has every cut
    u64 kept, there;
    m = sh.total;
    sort_list(m);
    list_sums(0);
    int cut = top_k && top_k < m ? top_k : m;
    if (min_p > 0.0f) {  // the items with w >= min_p come first
      if (tid == 0) sh.pick_count = 0;
      __syncthreads();
      int c = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int x = tid * kPer + i;
        c += x < m && rule.share(key_logit(static_cast<uint32_t>(items[x] >> kIndexBits))) >= min_share;
      }
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0 && c) atomicAdd(&sh.pick_count, c);
      __syncthreads();
      cut = min(cut, sh.pick_count);
    }
    share_item([&](int i) { return tid * kPer + i == cut - 1; }, &kept);
    if (top_p > 0.0f) {
      u64 z = 0;
      for (int c = 0; c < ctas; ++c) z += sh.whole[c];
      const u64 target = part_of(top_p, z);
      if (target < kept) {  // reached within the list
        reach(target, &there);
        kept = there;
      }
    }
    const int item = reach(part_of(u, kept), &there);
    answer(item, kept);
    cluster.barrier_wait();
    return;
  }

  // ---- 3. by the histogram
  u64 z = 0, kept = 0, tokens = 0;
  {
    // Every CTA finds the steps of the cuts and, as those bound what is kept from both
    // sides, the one or two steps the draw can be in; all are listed at once.
    constexpr int kOwn = kBins / kThreads;
    u64 mass[kOwn], mine = 0;
    uint32_t count[kOwn], mine_n = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      mass[i] = tot_mass[tid * kOwn + i];
      count[i] = top_k ? tot_count[tid * kOwn + i] : 0;
      mine += mass[i];
      mine_n += count[i];
    }
    const u64 upto = block_scan(mine, sh.red), upto_n = top_k ? block_scan(mine_n, sh.red) : 0;
    if (tid == kThreads - 1) {
      sh.sum = upto;
      sh.tokens = upto_n;
    }
    __syncthreads();
    z = sh.sum;
    tokens = sh.tokens;
    if (min_p > 0.0f)
      for (int c = 0; c < ctas; ++c) kept += sh.above[c];
    else
      kept = z;
    auto locate = [&](int which, bool by_count, u64 target) {
      u64 at = upto - mine, at_n = upto_n - mine_n;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const u64 has = by_count ? at_n : at, gets = has + (by_count ? count[i] : mass[i]);
        if (has < target && gets >= target) {
          Step &t = sh.step[which];
          t.bin = tid * kOwn + i;
          t.before = at;
          t.mass = mass[i];
          t.before_n = static_cast<int>(at_n);
          t.count = static_cast<int>(count[i]);
        }
        at += mass[i];
        at_n += count[i];
      }
    };
    const u64 cut = top_p > 0.0f ? part_of(top_p, z) : kept;
    const bool cuts_p = cut < kept, cuts_k = top_k && static_cast<u64>(top_k) < tokens;
    if (cuts_p) locate(0, false, cut);
    if (cuts_k) locate(1, true, top_k);
    __syncthreads();
    const Step sp = sh.step[0], sk = sh.step[1];
    u64 fewest = kept, most = kept;
    if (cuts_p) {
      fewest = cut;
      most = min(most, sp.before + sp.mass);
    }
    if (cuts_k) {
      fewest = min(fewest, sk.before + 1);
      most = min(most, sk.before + sk.mass);
    }
    locate(2, false, part_of(u, fewest));
    locate(3, false, part_of(u, most));
    __syncthreads();
    const Step s0 = sh.step[2], s1 = sh.step[3];
    // the cuts' steps that lie behind the draw's, in order (kBins: none)
    int c0 = cuts_p && sp.bin > s1.bin ? sp.bin : kBins, c1 = cuts_k && sk.bin > s1.bin && sk.bin != c0 ? sk.bin : kBins;
    if (c1 < c0) {
      const int t = c0;
      c0 = c1;
      c1 = t;
    }
    const int last = c1 < kBins ? c1 : c0 < kBins ? c0 : s1.bin;
    gather(under_step(last), over_step(s0.bin), [&](float l, int) {
      const int b = rule.bin(l);
      return (b >= s0.bin && b <= s1.bin) || b == c0 || b == c1;
    });
    cluster.sync();
    const bool overflow = first->total > kListCap;
    cluster.barrier_arrive();  // the first CTA outlives the others' look at its memory
    if (!overflow) {
      if (rank != 0) return;
      m = sh.total;
      sort_list(m);
      list_sums(s0.before);
      // a cut's step that lies apart goes on from its own sum and count
      const u64 end = s1.before + s1.mass;
      const int end_n = s1.before_n + s1.count;
      const Step &t0 = cuts_p && c0 == sp.bin ? sp : sk, &t1 = cuts_p && c1 == sp.bin ? sp : sk;
      int skipped[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int x = tid * kPer + i;
        skipped[i] = s0.before_n;
        if (x < m) {
          const int b = rule.bin(key_logit(static_cast<uint32_t>(items[x] >> kIndexBits)));
          if (b > s1.bin) {
            sums[i] += t0.before - end;
            skipped[i] += t0.before_n - end_n;
          }
          if (b > c0) {
            sums[i] += t1.before - (t0.before + t0.mass);
            skipped[i] += t1.before_n - (t0.before_n + t0.count);
          }
        }
      }
      u64 there;
      if (cuts_k) {
        share_item([&](int i) { return tid * kPer + i < m && tid * kPer + i + 1 + skipped[i] == top_k; }, &there);
        kept = min(kept, there);
      }
      if (cuts_p) {
        reach(cut, &there);
        kept = min(kept, there);
      }
      const int item = reach(part_of(u, kept), &there);
      answer(item, kept);
      cluster.barrier_wait();
      return;
    }
    cluster.barrier_wait();
  }

  // ---- otherwise the first CTA decides, the others gather and divide as it says
  // the tokens of a command's steps and range
  auto in_command = [&](const Command &c, float l, int j) {
    const int b = rule.bin(l);
    if (b < c.bin0 || b > c.bin1 || !(l > -INFINITY)) return false;
    const u64 o = token_ord(order_key(l), j);
    return o >= c.lo && o <= c.hi;
  };
  auto obey = [&]() -> bool {  // every CTA: false when the row is done
    cluster.sync();  // the command stands, the list is empty
    const Command c = first->cmd;
    if (c.op == kDone) {
      cluster.sync();  // the first CTA outlives the others' look at its memory
      return false;
    }
    if (c.op == kGather) {
      gather(-FLT_MAX, INFINITY, [&](float l, int j) { return in_command(c, l, j); });
    } else {
      for (int b = tid; b < 3 * kBins; b += kThreads) bin_count[b] = 0;
      __syncthreads();
      each([&](const float *l, int j) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          if (!in_command(c, l[i], j + i)) continue;
          const u64 w[1] = {rule.weight(l[i])}, s = (c.hi - token_ord(order_key(l[i]), j + i)) >> c.shift;
          const int b[1] = {static_cast<int>(min(s, (u64)(kBins - 1)))};
          const bool counts[1] = {w[0] != 0};
          count_in(w, b, counts, std::true_type());
        }
      });
      collect(list, reinterpret_cast<uint32_t *>(list + kBins), 1);
    }
    cluster.sync();
    return true;
  };
  if (rank != 0) {
    while (obey()) {
    }
    return;
  }
  // The step of `mass` / `count` in which the measure reaches target, from `before`
  // (sums) and `before_n` (tokens) on; a target outside what the steps hold (which sums
  // that agree rule out) is the first or the last of them.
  auto find_step = [&](const u64 *mass, const uint32_t *count, bool by_count, u64 target, u64 before, u64 before_n) {
    u64 m[kBins / kThreads], c[kBins / kThreads], ms = 0, cs = 0;
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      m[i] = mass[tid * (kBins / kThreads) + i];
      c[i] = count[tid * (kBins / kThreads) + i];
      ms += m[i];
      cs += c[i];
    }
    u64 all_m, all_c;
    u64 am = before + block_scan(ms, sh.red, &all_m) - ms;
    u64 ac = before_n + block_scan(cs, sh.red, &all_c) - cs;
    const u64 from = by_count ? before_n : before, all = by_count ? all_c : all_m;
    target = min(max(target, from + 1), from + max(all, 1ull));
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) {
      const u64 has = by_count ? ac : am, gets = has + (by_count ? c[i] : m[i]);
      if (has < target && gets >= target) {  // one step of the row
        sh.pick_bin = tid * (kBins / kThreads) + i;
        sh.pick_before = am;
        sh.pick_before_count = ac;
        sh.pick_count = static_cast<int>(c[i]);
      }
      am += m[i];
      ac += c[i];
    }
    __syncthreads();
  };
  // Lists the tokens around where the measure reaches target; returns the item there,
  // *sum_there the row's sum up to and with it.  If all tokens up to there fit the
  // list, they are listed and *from_start is set.
  auto select = [&](bool by_count, u64 target, bool *from_start, u64 *sum_there) __attribute__((always_inline)) {
    find_step(tot_mass, tot_count, by_count, target, 0, 0);
    Command c{};
    c.bin0 = c.bin1 = sh.pick_bin;
    c.hi = ~0ull;
    u64 before = sh.pick_before, before_n = sh.pick_before_count;
    int here = sh.pick_count;
    *from_start = top_k && before_n + here <= kListCap;
    if (*from_start) {
      c.bin0 = 0;
      before = before_n = 0;
      here = 0;
    }
    __syncthreads();
    // List the step's tokens, or divide it by ord until they fit (the counts, kept for a
    // top_k only, save an attempt).  ord has 52 bits and each division takes 10 of
    // them, after a first one by a range estimated from the step's logits (its last
    // part takes what lies below the estimate): 7 suffice.
    for (int level = 0; level < 9; ++level) {
      if (here <= kListCap) {
        c.op = kGather;
        if (tid == 0) {
          sh.cmd = c;
          sh.total = 0;
        }
        __syncthreads();
        obey();
        if (sh.total <= kListCap) break;
      }
      *from_start = false;  // tokens of no weight, which are not counted, did not fit
      if (level == 0) {
        const float w = rule.bin_scale > 0.0f ? 1.0f / rule.bin_scale : INFINITY;
        const uint32_t kh = order_key(high - w * static_cast<float>(c.bin0 - 1));  // over the step
        const uint32_t kl = order_key(high - w * static_cast<float>(c.bin0 + 1)), k0 = order_key(low);
        c.hi = c.bin0 == 0 || kh == 0 ? top : token_ord(kh, 0);
        const u64 lo = c.bin0 + 1 == kBins || kl < k0 ? static_cast<u64>(k0) << kIndexBits : token_ord(kl, (1 << kIndexBits) - 1);
        c.shift = 0;
        while (c.hi > lo && ((c.hi - lo) >> c.shift) >= kBins) ++c.shift;
      }
      c.op = kDivide;
      if (tid == 0) sh.cmd = c;
      __syncthreads();
      obey();
      find_step(list, reinterpret_cast<const uint32_t *>(list + kBins), by_count, target, before, before_n);
      const u64 s = sh.pick_bin;
      before = sh.pick_before;
      before_n = sh.pick_before_count;
      here = sh.pick_count;
      __syncthreads();
      c.hi -= s << c.shift;
      if (s + 1 < kBins) c.lo = c.hi - ((1ull << c.shift) - 1);  // the last step runs down to lo
      const u64 size = c.hi - c.lo;
      c.shift = 0;
      while ((size >> c.shift) >= kBins) ++c.shift;
    }
    m = min(sh.total, kListCap);
    sort_list(m);
    list_sums(before);
    if (by_count) {
      const int item = min(static_cast<int>(target - before_n) - 1, m - 1);
      return share_item([&](int i) { return tid * kPer + i == item; }, sum_there);
    }
    return reach(target, sum_there);
  };
  bool from_start = false;
  u64 there;
  if (top_k && static_cast<u64>(top_k) < tokens) {
    select(true, top_k, &from_start, &there);
    kept = min(kept, there);
  }
  if (top_p > 0.0f) {
    const u64 target = part_of(top_p, z);
    if (target < kept) {
      if (from_start)
        reach(target, &there);
      else
        select(false, target, &from_start, &there);
      kept = min(kept, there);
    }
  }
  const u64 target = part_of(u, kept);
  int item;
  if (from_start)
    item = reach(target, &there);
  else
    item = select(false, target, &from_start, &there);
  answer(item, kept);
  __syncthreads();
  if (tid == 0) sh.cmd.op = kDone;
  __syncthreads();
  obey();
}


// ------------------------------------------------------------- bf16 rows
// A bf16 row has few distinct values, so a histogram of the values themselves needs
// one 32-bit count a token and no exponential: the sum of w of a value is its
// count times its w.  The cuts and the draw find their value by prefix sums, and
// a tie is settled by counting in index order: no list, no sort.
//
// The histogram spans the 2048 magnitudes (16 binades) below the larger of |max l|
// and |max(min l, max l - 36 T)| for either sign; what is lower has weights that
// round to nothing.  Zero has a place of its own; the few logits nearer to it than the
// span's least (2^-16 of the largest) share one place a sign, their sums formed
// token by token, and a cut or draw that falls there is found by a slow search
// (rows of nothing but such logits aside, about one in 10^4).  An f16 row has
// eight times the values: it goes with the f32 ones.
//
// Measured: 256 rows of 128256 with nucleus, min-p and plain settings (65.7 MB, 10.2 us at
// a plain copy's rate) 62.9 us.  Leaving parts out of a slightly slower form: the two readings
// and the maximum 15, forming the indices 15, the shared atomics 26 (8 were no two of a
// warp to meet in a bank), the cuts and the draw 11.  The rows are read from DRAM once (65.9 MB), then from L2.
constexpr int kVals = 2048;
// places, in falling order of their logits
constexpr int kTinyPos = kVals, kZeroAt = kVals + 1, kTinyNeg = kVals + 2, kNeg0 = kVals + 3;
constexpr int kPlaces = 2 * kVals + 3;
constexpr int kValueThreads = 512;
// Vectors of 16 bytes a thread has in flight while it counts as many: 256 rows of 128256 take
// 62.9 us with 2, 67.6 with 3 (registers spill).
constexpr int kAhead = 2;

// Where a place is counted: positive magnitudes upwards, then negative ones upwards
// and the three about zero, so that a token's index is its bits and one product away.
__device__ __forceinline__ int count_index(int place) {
  return place < kVals ? kVals - 1 - place : place >= kNeg0 ? kVals + place - kNeg0 : 2 * kVals + place - kTinyPos;
}

struct ValueShared {
  double tab[kExpTable];
  u64 red[kValueThreads / 32];
  float warp_high[kValueThreads / 32], warp_low[kValueThreads / 32];
  // written by every CTA of the row into every other
  float high[kMaxCluster], low[kMaxCluster];
  u64 mass[kMaxCluster], count[kMaxCluster], above[kMaxCluster];
  // of this CTA: the places that counters keep (kTinyPos, kZeroAt, kTinyNeg)
  u64 tiny_mass[3], tiny_above[3];
  // what the owner of a cut's place tells (top_k's, top_p's, the draw's)
  struct {
    int place;
    u64 before, before_n;
  } told[3];
  u64 bins[256];
  u64 pick[2];
};

template <int NT>
__device__ __forceinline__ u64 block_sum_n(u64 v, u64 *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) v += red[w];
  return v;
}

__device__ __forceinline__ float bf16_bits(uint32_t b) { return __uint_as_float(b << 16); }

// Logits before the first on 16 bytes.
__device__ __forceinline__ int to_vector(const unsigned short *row) {
  return static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / 2);
}

__global__ void __launch_bounds__(kValueThreads, 2) k_sample_values(const RowArgs p) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  __shared__ ValueShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int own = (kPlaces + ctas - 1) / ctas, p0 = rank * own, p1 = min(kPlaces, p0 + own);  // the places this CTA sums
  uint32_t *count = reinterpret_cast<uint32_t *>(s_dyn);  // [kPlaces], of this CTA's tokens
  u64 *mass = reinterpret_cast<u64 *>(count + (kPlaces + 3) / 4 * 4);  // [own], of the row
  uint32_t *total = reinterpret_cast<uint32_t *>(mass + own);          // [own], of the row
  const LlmqSampleRows &a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / ctas, j0 = rank * p.slice, n = max(0, min(p.slice, a.vocab - j0));
  cluster.barrier_arrive();
  if (tid < kExpTable) sh.tab[tid] = exp2(p.scale - tid * (1.0 / kExpTable));
  if (tid < 3) sh.tiny_mass[tid] = sh.tiny_above[tid] = 0;
  for (int i = tid; i < kPlaces; i += kValueThreads) count[i] = 0;
  serve_wait();
  serve_dependents();
  const unsigned short *whole_row = static_cast<const unsigned short *>(a.logits) + r * a.stride, *row = whole_row + j0;
  const float temp = a.temperature ? a.temperature[r] : 1.0f;
  const bool greedy = !(temp > 0.0f);
  const float min_p = a.min_p && a.min_p[r] > 0.0f ? fminf(a.min_p[r], 1.0f) : 0.0f;
  const float top_p = a.top_p && a.top_p[r] > 0.0f && a.top_p[r] < 1.0f ? a.top_p[r] : 0.0f;
  const int top_k = a.top_k && a.top_k[r] > 0 && a.top_k[r] < a.vocab ? a.top_k[r] : 0;

  // ---- the largest and least logit (of two at a time; NaN is passed over)
  float high = -INFINITY, low = INFINITY;
  {
    const __nv_bfloat162 nan = __floats2bfloat162_rn(NAN, NAN);
    __nv_bfloat162 hi2 = nan, lo2 = nan;
    const int head = min(n, to_vector(row)), nv = (n - head) / 8;
    const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
    auto add2 = [&](uint32_t w) {
      const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162 *>(&w);
      hi2 = __hmax2(hi2, x);
      lo2 = __hmin2(lo2, x);
    };
    for (int v = tid; v < nv; v += 8 * kValueThreads) {
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = v + i * kValueThreads < nv ? vec[v + i * kValueThreads] : make_uint4(~0u, ~0u, ~0u, ~0u);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        add2(x[i].x);
        add2(x[i].y);
        add2(x[i].z);
        add2(x[i].w);
      }
    }
    for (int e = tid; e < n - 8 * nv; e += kValueThreads) {  // the ends
      const float l = bf16_bits(row[e < head ? e : e + 8 * nv]);
      high = fmaxf(high, l);
      low = fminf(low, l);
    }
    high = fmaxf(high, fmaxf(__low2float(hi2), __high2float(hi2)));
    low = fminf(low, fminf(__low2float(lo2), __high2float(lo2)));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if (lane == 0) {
    sh.warp_high[warp] = high;
    sh.warp_low[warp] = low;
  }
  __syncthreads();
  cluster.barrier_wait();
  if (tid < ctas) {
    for (int w = 0; w < kValueThreads / 32; ++w) {
      high = fmaxf(high, sh.warp_high[w]);
      low = fminf(low, sh.warp_low[w]);
    }
    ValueShared *to = cluster.map_shared_rank(&sh, tid);
    to->high[rank] = high;
    to->low[rank] = low;
  }
  cluster.sync();
  for (int c = 0; c < ctas; ++c) {
    high = fmaxf(high, sh.high[c]);
    low = fminf(low, sh.low[c]);
  }
  if (high == -INFINITY) {  // nothing can be drawn
    if (rank == 0 && tid == 0) {
      a.ids[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  RowRule rule;
  rule.set(high, temp, p.scale, sh.tab);
  const double min_share = static_cast<double>(min_p) * static_cast<double>(1ull << p.scale);
  // the span's least magnitude
  const float far = fmaxf(fabsf(high), greedy ? 0.0f : fabsf(fmaxf(low, high - 36.0f * temp)));
  const int least = min(max(static_cast<int>(__float_as_uint(far) >> 16) + 1 - kVals, 1), 0x7f81 - kVals);
  auto value_at = [&](int place) -> float {  // a place of one value
    if (place < kVals) return bf16_bits(least + kVals - 1 - place);
    return place >= kNeg0 ? bf16_bits((least + place - kNeg0) | 0x8000u) : 0.0f;
  };
  auto one_value = [&](int place) { return place != kTinyPos && place != kTinyNeg; };
  int place = 0;
  u64 nth = 1, kept = 0;
  if (greedy) {
    place = high == 0.0f ? kZeroAt : high > 0.0f ? kVals - 1 + least - static_cast<int>(__float_as_uint(high) >> 16)
                                                 : kNeg0 + static_cast<int>((__float_as_uint(high) >> 16) & 0x7fffu) - least;
  }

  // ---- counts of values, without a branch: the byte offset of a token's count is
  // 4 (magnitude - least) + (negative ? 4 kVals : 0), and 4 kVals is its sign bit / 4
  static_assert(4 * kVals == 0x8000 / 4, "the sign bit moves to its offset");
  const uint32_t counts = static_cast<uint32_t>(__cvta_generic_to_shared(count));
  uint32_t zeros = 0, pos_n = 0, neg_n = 0;
  u64 pos_m = 0, neg_m = 0, pos_a = 0, neg_a = 0;
  auto add = [&](uint32_t mag, uint32_t sign) -> int {  // sign: in bit 15
    const int x = static_cast<int>(mag) - least;
    // what lies past the span is too low to count, -infinity or NaN
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.lt.u32 q, %0, %1;\n\t@q red.shared.add.u32 [%2], 1;\n\t}" ::"r"(x), "n"(kVals),
        "r"(counts + 4 * x + ((sign >> 2) & 0x2000u))
        : "memory");
    return x;  // below 0: nearer to zero than the span
  };
  auto add2 = [&](uint32_t w) -> int {
    const uint32_t m = w & 0x7fff7fffu;
    return add(m & 0xffffu, w) | add(m >> 16, w >> 16);
  };
  auto add_near = [&](uint32_t b) {
    const int mag = b & 0x7fff;
    if (mag >= least) return;
    if (mag == 0) {
      ++zeros;
      return;
    }
    const RowRule::Product e = rule.product_any(bf16_bits(b));
    const u64 w = rule.weight(e), v = rule.share(e) >= min_share ? w : 0;
    if (b & 0x8000u) {
      ++neg_n;
      neg_m += w;
      neg_a += v;
    } else {
      ++pos_n;
      pos_m += w;
      pos_a += v;
    }
  };
  {
    const int head = min(n, to_vector(row)), nv = (n - head) / 8;
    const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
    uint4 x[kAhead], next[kAhead];
    auto fetch = [&](int v) {  // what is past the end counts as NaN
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        next[i] = v + i * kValueThreads < nv ? vec[v + i * kValueThreads] : make_uint4(~0u, ~0u, ~0u, ~0u);
    };
    fetch(tid);
    for (int v = tid; v < nv; v += kAhead * kValueThreads) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = next[i];
      fetch(v + kAhead * kValueThreads);
      int near = 0;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) near |= add2(x[i].x) | add2(x[i].y) | add2(x[i].z) | add2(x[i].w);
      if (near < 0) {  // seldom: look at them again (reading them again, one by one, took 3 us more)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {  // (what is past the end is NaN: passed over)
          const uint4 y = x[i];
#pragma unroll 1
          for (int e = 0; e < 8; ++e)
            add_near(((e < 4 ? e < 2 ? y.x : y.y : e < 6 ? y.z : y.w) >> (16 * (e & 1))) & 0xffffu);
        }
      }
    }
#pragma unroll 1
    for (int e = tid; e < n - 8 * nv; e += kValueThreads) {  // the ends
      const uint32_t b = row[e < head ? e : e + 8 * nv];
      if (add(b & 0x7fffu, b) < 0) add_near(b);
    }
  }
  if (zeros) atomicAdd(&count[count_index(kZeroAt)], zeros);
  if (pos_n) {
    atomicAdd(&count[count_index(kTinyPos)], pos_n);
    atomicAdd(&sh.tiny_mass[0], pos_m);
    atomicAdd(&sh.tiny_above[0], pos_a);
  }
  if (neg_n) {
    atomicAdd(&count[count_index(kTinyNeg)], neg_n);
    atomicAdd(&sh.tiny_mass[2], neg_m);
    atomicAdd(&sh.tiny_above[2], neg_a);
  }
  cluster.sync();

  if (!greedy) {
    // ---- each CTA sums its places over the cluster, a thread `per` adjacent ones (odd: no
    // two lanes of a warp in one bank)
    for (int i = p0 + tid; i < p1; i += kValueThreads) {
      const int at = count_index(i);
      uint32_t c = 0;
      for (int q = 0; q < ctas; ++q) c += cluster.map_shared_rank(count, q)[at];
      total[i - p0] = c;
    }
    __syncthreads();
    const int per = ((own + kValueThreads - 1) / kValueThreads) | 1;
    const int i0 = min(p1 - p0, tid * per), i1 = min(p1 - p0, i0 + per);
    u64 mine_m = 0, mine_n = 0, mine_a = 0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t c = total[i];
      u64 m = 0, v = 0;
      if (c && one_value(p0 + i)) {
        const RowRule::Product e = rule.product_any(value_at(p0 + i));
        m = c * rule.weight(e);
        v = rule.share(e) >= min_share ? m : 0;
      } else if (c) {
        for (int q = 0; q < ctas; ++q) {
          const ValueShared *o = cluster.map_shared_rank(&sh, q);
          m += o->tiny_mass[p0 + i - kTinyPos];
          v += o->tiny_above[p0 + i - kTinyPos];
        }
      }
      mass[i] = m;
      mine_m += m;
      mine_n += c;
      mine_a += v;
    }
    // sums and counts up to and with each thread's places
    const u64 upto_m = block_scan<kValueThreads>(mine_m, sh.red);
    const u64 upto_n = top_k ? block_scan<kValueThreads>(mine_n, sh.red) : 0;
    if (min_p > 0.0f) mine_a = block_sum_n<kValueThreads>(mine_a, sh.red);
    if (tid == kValueThreads - 1)
      for (int q = 0; q < ctas; ++q) {
        ValueShared *to = cluster.map_shared_rank(&sh, q);
        to->mass[rank] = upto_m;
        to->count[rank] = upto_n;
        to->above[rank] = mine_a;
      }
    cluster.sync();
    u64 z = 0, usable = 0, above = 0;
    for (int c = 0; c < ctas; ++c) {
      z += sh.mass[c];
      usable += sh.count[c];
      above += sh.above[c];
    }
    kept = min_p > 0.0f ? above : z;

    // Every CTA: the place where the measure (counts or sums) reaches target, and both up
    // to it.  The CTA that owns the place tells the others.
    u64 before = 0, before_n = 0;
    auto find = [&](int which, bool by_count, u64 target) {
      u64 bm = 0, bn = 0;
      int owner = 0;
      for (; owner + 1 < ctas; ++owner) {
        if ((by_count ? bn + sh.count[owner] : bm + sh.mass[owner]) >= target) break;
        bm += sh.mass[owner];
        bn += sh.count[owner];
      }
      if (owner == rank) {
        u64 am = bm + upto_m - mine_m, ac = by_count ? bn + upto_n - mine_n : 0;
        if ((by_count ? ac : am) < target && (by_count ? ac + mine_n : am + mine_m) >= target) {  // one thread
          int i = i0;
          for (; (by_count ? ac + total[i] : am + mass[i]) < target; ++i) {
            am += mass[i];
            ac += total[i];
          }
          for (int q = 0; q < ctas; ++q) {
            auto *to = &cluster.map_shared_rank(&sh, q)->told[which];
            to->place = p0 + i;
            to->before = am;
            to->before_n = ac;
          }
        }
      }
      cluster.sync();
      place = sh.told[which].place;
      before = sh.told[which].before;
      before_n = sh.told[which].before_n;
    };
    // Within a place of many values, from `before` on: the key and what precedes it, by
    // every CTA alone over the whole row (slow; see above)
    uint32_t key = 0;
    auto find_tiny = [&](bool by_count, u64 target) {
      const bool neg = place == kTinyNeg;
      uint32_t prefix = 0, mask = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = tid; i < 256; i += kValueThreads) sh.bins[i] = 0;
        __syncthreads();
        for (int j = tid; j < a.vocab; j += kValueThreads) {
          const uint32_t b = whole_row[j];
          const int mag = b & 0x7fff;
          const uint32_t k = order_key(bf16_bits(b));
          if (mag > 0 && mag < least && static_cast<bool>(b & 0x8000u) == neg && (k & mask) == prefix)
            atomicAdd(&sh.bins[(k >> shift) & 255u], by_count ? 1ull : rule.weight(bf16_bits(b)));
        }
        __syncthreads();
        if (tid == 0) {
          u64 at = by_count ? before_n : before;
          int d = 255;
          for (; d > 0 && at + sh.bins[d] < target; --d) at += sh.bins[d];
          sh.pick[0] = d;
          sh.pick[1] = at;
        }
        __syncthreads();
        (by_count ? before_n : before) = sh.pick[1];
        prefix |= static_cast<uint32_t>(sh.pick[0]) << shift;
        mask |= 255u << shift;
      }
      key = prefix;
      if (by_count) {  // the sum of what precedes the key
        u64 m = 0;
        for (int j = tid; j < a.vocab; j += kValueThreads) {
          const uint32_t b = whole_row[j];
          const int mag = b & 0x7fff;
          const float l = bf16_bits(b);
          if (mag > 0 && mag < least && static_cast<bool>(b & 0x8000u) == neg && order_key(l) > key) m += rule.weight(l);
        }
        before += block_sum_n<kValueThreads>(m, sh.red);
      }
    };
    auto reach = [&](int which, bool by_count, u64 target) -> u64 {  // its w
      find(which, by_count, target);
      if (!one_value(place)) {
        find_tiny(by_count, target);
        return rule.weight(key_logit(key));
      }
      return rule.weight(value_at(place));
    };
    if (top_k && static_cast<u64>(top_k) < usable) {
      const u64 w = reach(0, true, top_k);
      kept = min(kept, before + (top_k - before_n) * w);
    }
    if (top_p > 0.0f) {
      const u64 target = part_of(top_p, z);
      if (target < kept) {
        const u64 w = reach(1, false, target);
        kept = min(kept, before + (target - before + w - 1) / w * w);
      }
    }
    const float uf = a.u[r];
    const u64 target = part_of(uf > 0.0f ? fminf(uf, 1.0f) : 0.0f, kept);
    const u64 w = reach(2, false, target);
    nth = (target - before + w - 1) / w;
    if (!one_value(place)) {  // among all tokens of the row with this key, by the first CTA alone
      const uint32_t code = __float_as_uint(key_logit(key)) >> 16;
      if (rank == 0 && warp == 0) {
        u64 seen = 0;
        for (int j1 = 0; j1 < a.vocab && seen < nth; j1 += 32) {
          const unsigned bal = __ballot_sync(0xffffffffu, j1 + lane < a.vocab && whole_row[j1 + lane] == code);
          if (((bal >> lane) & 1u) && seen + __popc(bal & ((1u << lane) - 1u)) + 1 == nth) {
            a.ids[r] = j1 + lane;
            if (a.logprobs) {
              const double lw = -(rule.mxd - static_cast<double>(key_logit(key))) / static_cast<double>(temp);
              a.logprobs[r] = static_cast<float>(lw - log(ldexp(static_cast<double>(kept), -p.scale)));
            }
          }
          seen += __popc(bal);
        }
      }
      return;
    }
  }

  // ---- the nth token of the place's value, in index order
  int owner = 0;
  {
    const uint32_t c = lane < ctas ? cluster.map_shared_rank(count, lane)[count_index(place)] : 0;
    const u64 upto = warp_scan(c);
    const unsigned who = __ballot_sync(0xffffffffu, lane < ctas && upto >= nth);
    owner = __ffs(who) - 1;
    nth -= __shfl_sync(0xffffffffu, upto - c, owner & 31);
  }
  cluster.barrier_arrive();  // a CTA outlives the others' look at its counts
  if (owner == rank) {
    // each warp a part of the slice, 16 bytes a lane and step (+0 and -0 compare as equal)
    const float want = value_at(place);
    const uint32_t code = __float_as_uint(want) >> 16, ignore = place == kZeroAt ? 0x7fffu : 0xffffu;
    const int head = min(n, to_vector(row)), nv = (n - head) / 8, part = (nv + kValueThreads - 1) / kValueThreads * 32;
    const int va = min(nv, warp * part), vb = min(nv, va + part);
    const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
    const uint32_t code2 = code | (code << 16);
    auto hits = [&](uint32_t w) -> uint32_t {  // bit 0 and bit 16: the halves that match
      return __heq2_mask(*reinterpret_cast<const __nv_bfloat162 *>(&w), *reinterpret_cast<const __nv_bfloat162 *>(&code2)) &
             0x00010001u;
    };
    auto hits8 = [&](const uint4 x) { return hits(x.x) + hits(x.y) + hits(x.z) + hits(x.w); };
    uint32_t c2 = 0;  // two counts of at most 2^15 / 32 steps of 4
#pragma unroll 4
    for (int v = va + lane; v < vb; v += 32) c2 += hits8(vec[v]);
    int c = static_cast<int>((c2 & 0xffffu) + (c2 >> 16));
    c = __reduce_add_sync(0xffffffffu, c);
    // what does not fill a vector: the head before all, the tail behind all
    auto single = [&](int j) { return (row[j] & ignore) == code; };
    if (lane == 0) sh.red[warp] = c;
    const unsigned head_bal = __ballot_sync(0xffffffffu, lane < head && single(lane));
    __syncthreads();
    u64 seen = __popc(head_bal);
    auto tell = [&](int j) {
      a.ids[r] = j0 + j;
      if (a.logprobs) {
        const double lw = want == high ? 0.0 : -(rule.mxd - static_cast<double>(want)) / static_cast<double>(temp);
        a.logprobs[r] = greedy ? 0.0f : static_cast<float>(lw - log(ldexp(static_cast<double>(kept), -p.scale)));
      }
    };
    if (nth <= seen) {  // in the head
      if (warp == 0 && ((head_bal >> lane) & 1u) && __popc(head_bal & ((1u << lane) - 1u)) + 1 == nth) tell(lane);
    } else {
      for (int w = 0; w < warp; ++w) seen += sh.red[w];
      if (seen < nth && seen + c >= nth) {
        for (int v0 = va; v0 < vb && seen < nth; v0 += 32) {
          const int v = v0 + lane;
          const uint4 x = v < vb ? vec[v] : make_uint4(0, 0, 0, 0);
          const uint32_t h = v < vb ? hits8(x) : 0u;
          const int mine = static_cast<int>((h & 0xffffu) + (h >> 16));
          const int incl = static_cast<int>(warp_scan(mine));
          if (seen + incl >= nth && seen + incl - mine < nth) {
            int left = static_cast<int>(nth - seen) - (incl - mine), j = head + 8 * v;
            for (; left > 0; ++j) left -= single(j);
            tell(j - 1);
          }
          seen += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
      if (warp == kValueThreads / 32 - 1 && seen + c < nth) {  // in the tail
        const int j = head + 8 * nv + lane;
        const unsigned bal = __ballot_sync(0xffffffffu, j < n && single(j));
        if (((bal >> lane) & 1u) && seen + c + __popc(bal & ((1u << lane) - 1u)) + 1 == nth) tell(j);
      }
    }
  }
  cluster.barrier_wait();
}

inline int scale_bits(int vocab) {
  int log2v = 0;
  while ((1 << log2v) < vocab) ++log2v;
  return 62 - log2v < 50 ? 62 - log2v : 50;
}

// A launch of n_rows clusters of `ctas` CTAs, with programmatic dependent launch.  The
// kernel's limit is set to the most any call takes, so that calls from several threads
// do not lower it for one another.
cudaError_t launch_clusters(void (*kern)(RowArgs), const RowArgs &p, int ctas, int threads, int smem, int most,
                            cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.a.n_rows) * ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  llmqd_count_launch();
  return cudaLaunchKernelEx(&cfg, kern, p);
}

cudaError_t launch_values(const LlmqSampleRows &a, int sms, cudaStream_t st) {
  RowArgs p{};
  p.a = a;
  p.scale = scale_bits(a.vocab);
  // CTAs a row until every SM has one (rows of 128256): 128 rows 38 us in clusters of 2, 44
  // alone, 45 of 4; 256 rows 63 us alone, 68 in clusters of 2
  int ctas = 1;
  while (ctas < kMaxCluster && (long long)a.n_rows * ctas < sms && a.vocab / ctas > 4 * kValueThreads) ctas *= 2;
  p.slice = ((a.vocab + ctas - 1) / ctas + 15) / 16 * 16;
  const int own = (kPlaces + ctas - 1) / ctas;
  const int smem = (kPlaces + 3) / 4 * 16 + own * 12;
  return launch_clusters(k_sample_values, p, ctas, kValueThreads, smem, (kPlaces + 3) / 4 * 16 + kPlaces * 12, st);
}

template <typename T>
cudaError_t launch(const LlmqSampleRows &a, int sms, cudaStream_t st) {
  RowArgs p{};
  p.a = a;
  p.scale = scale_bits(a.vocab);
  // CTAs a row: as many as let all rows be on the GPU at once, two CTAs an SM.  (64 rows of
  // 128256 f32 logits, top-k 50: 24 us in clusters of 4, 35 us of 8, which take two turns,
  // 31 of 2.)
  int ctas = 1;
  auto slice_of = [&](int c) { return ((a.vocab + c - 1) / c + 15) / 16 * 16; };
  while (ctas < kMaxCluster && 2LL * a.n_rows * ctas <= 2 * sms && slice_of(ctas) > 2 * kThreads) ctas *= 2;
  p.slice = slice_of(ctas);
  p.resident = p.slice * sizeof(T) <= kMaxResident;  // beyond, two CTAs' slices do not fit an SM: from L2 each time
  const int smem = kWorkBytes + (p.resident ? p.slice * (int)sizeof(T) : 0);
  return launch_clusters(k_sample_rows<T>, p, ctas, kThreads, smem, kWorkBytes + kMaxResident, st);
}

}  // namespace

extern "C" LLMQ_API int llmq_sample_rows(const LlmqSampleRows *a, void *stream) {
  ServeCheck c("llmq_sample_rows");
  c.require(a != nullptr, "null descriptor");
  if (c.rc != LLMQ_OK) return c.rc;
  c.require(serve_dtype(a->dtype), "unknown type of the logits");
  c.require(a->n_rows >= 0 && a->n_rows <= INT_MAX / kMaxCluster, "n_rows outside 0..2^28 - 1");
  c.require(a->vocab > 0 && a->vocab <= (1 << kIndexBits), "vocab outside 1..2^20");
  if (c.rc != LLMQ_OK || a->n_rows == 0) return c.rc;
  c.require(a->logits && a->u && a->ids, "null pointer");
  c.require(a->stride >= a->vocab, "a row stride is shorter than its row");
  c.require(aligned_to(a->logits, serve_bytes(a->dtype)), "the logits do not start on an element");
  c.elements(a->temperature, "temperature");
  c.elements(a->top_k, "top_k");
  c.elements(a->top_p, "top_p");
  c.elements(a->min_p, "min_p");
  c.elements(a->u, "u");
  c.elements(a->ids, "ids");
  c.elements(a->logprobs, "logprobs");
  c.on_device();
  c.memory(a->logits, "logits");
  c.memory(a->temperature, "temperature");
  c.memory(a->top_k, "top_k");
  c.memory(a->top_p, "top_p");
  c.memory(a->min_p, "min_p");
  c.memory(a->u, "u");
  c.memory(a->ids, "ids");
  c.memory(a->logprobs, "logprobs");
  if (c.rc != LLMQ_OK) return c.rc;
  int sms = 0;
  c.launched(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c.device));
  if (c.rc != LLMQ_OK) return c.rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  c.launched(a->dtype == LLMQ_F32   ? launch<float>(*a, sms, st)
             : a->dtype == LLMQ_F16 ? launch<__half>(*a, sms, st)
                                    : launch_values(*a, sms, st));
  return c.rc;
}
