// llmq_sample_rows.cu - one token for each row of a batch of logits, by
// temperature, top-k, min-p and top-p, from given random numbers
// (llmq_sample_rows).
//
// A row's weights are w_j = exp((l_j - max l) / T), as 64-bit integers: w_j is
// rounded to a whole number of 2^-S, S = 62 - ceil(log2 vocab), so any sum
// of them is exact, fits 63 bits and is the same in any order.  The tokens'
// order is the logit's bits mapped to an unsigned key of the same order (key 0:
// NaN and -infinity, never drawn), then the index.  Each of the three cuts keeps
// a prefix of that order, so what is kept is known by its sum alone; the draw is
// the first token at which the sum reaches u times the kept one.
#include <climits>
#include <cmath>

#include "llmq_serve.cuh"

using namespace llmq;

namespace {

constexpr int kThreads = 1024;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __float_as_uint(__fadd_rn(l, 0.0f));  // -0 to +0: equal logits, equal keys
  if (!(l > -INFINITY)) return 0u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

struct RowRule {
  float mx;       // the largest logit
  double inv_t;
  double one;     // 2^S
  // w of a token that is not excluded (0 beside an infinite maximum, whatever T)
  __device__ __forceinline__ double share(float l) const {
    return l == mx ? 1.0 : mx == INFINITY ? 0.0 : exp((static_cast<double>(l) - static_cast<double>(mx)) * inv_t);
  }
  __device__ __forceinline__ u64 weight(float l) const {
    return __double2ull_rn(share(l) * one);
  }
};

template <typename V>
__device__ __forceinline__ V block_sum(V v, V *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Found {
  uint32_t key;
  u64 before;  // measure of the tokens with larger keys
};

// The key at which the measure (1 or w of each token, over falling keys) reaches
// `target` (1 .. the row's whole measure): four levels of 256 bins.
template <bool mass, typename T>
__device__ Found reach(const T *row, int V, const RowRule &rule, u64 target, u64 *bins, u64 *pick) {
  uint32_t prefix = 0u, mask = 0u;
  u64 before = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int b = threadIdx.x; b < 256; b += kThreads) bins[b] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < V; j += kThreads) {
      const float l = to_f32(row[j]);
      const uint32_t k = order_key(l);
      if (k != 0u && (k & mask) == prefix) atomicAdd(&bins[(k >> shift) & 255u], mass ? rule.weight(l) : 1ull);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int b = 255;
      u64 sum = before;
      for (; b > 0 && sum + bins[b] < target; --b) sum += bins[b];
      pick[0] = b;
      pick[1] = sum;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(pick[0]) << shift;
    before = pick[1];
    mask |= 255u << shift;
  }
  return Found{prefix, before};
}

// ceil(f * total) in 1 .. total
__device__ __forceinline__ u64 part_of(double f, u64 total) {
  const double t = ceil(f * static_cast<double>(total));
  const u64 v = t < 1.0 ? 1ull : static_cast<u64>(t);
  return v > total ? total : v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_rows(const LlmqSampleRows a, int bits) {
  __shared__ u64 s_bins[256], s_red[32], s_pick[2];
  __shared__ uint32_t s_key[32];
  __shared__ int s_idx[32];
  serve_wait();
  serve_dependents();
  const int r = blockIdx.x, V = a.vocab, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *row = static_cast<const T *>(a.logits) + r * a.stride;
  // the first largest logit
  uint32_t best = 0u;
  int at = INT_MAX;
  for (int j = tid; j < V; j += kThreads) {
    const uint32_t k = order_key(to_f32(row[j]));
    if (k > best) {
      best = k;
      at = j;
    }
  }
  auto better = [&](uint32_t k, int i) {
    if (k > best || (k == best && i < at)) {
      best = k;
      at = i;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t k = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    better(k, i);
  }
  if (lane == 0) {
    s_key[warp] = best;
    s_idx[warp] = at;
  }
  __syncthreads();
  for (int w = 0; w < 32; ++w) better(s_key[w], s_idx[w]);
  const float temp = a.temperature ? a.temperature[r] : 1.0f;
  if (best == 0u || !(temp > 0.0f)) {
    if (tid == 0) {
      a.ids[r] = best == 0u ? -1 : at;
      if (a.logprobs) a.logprobs[r] = best == 0u ? -INFINITY : 0.0f;
    }
    return;
  }
  RowRule rule{key_logit(best), 1.0 / static_cast<double>(temp), ldexp(1.0, bits)};
  const float min_p = a.min_p && a.min_p[r] > 0.0f ? fminf(a.min_p[r], 1.0f) : 0.0f, top_p = a.top_p ? a.top_p[r] : 0.0f;
  const int top_k = a.top_k ? a.top_k[r] : 0;
  // the whole sum, the sum of w >= min_p, the number of tokens that can be drawn
  u64 whole = 0, above = 0, count = 0;
  for (int j = tid; j < V; j += kThreads) {
    const float l = to_f32(row[j]);
    if (order_key(l) == 0u) continue;
    const double e = rule.share(l);
    const u64 w = __double2ull_rn(e * rule.one);
    whole += w;
    above += min_p > 0.0f && !(e >= static_cast<double>(min_p)) ? 0 : w;
    ++count;
  }
  whole = block_sum(whole, s_red);
  above = block_sum(above, s_red);
  count = block_sum(count, s_red);
  u64 kept = above;
  if (top_k > 0 && static_cast<u64>(top_k) < count) {
    const Found f = reach<false>(row, V, rule, top_k, s_bins, s_pick);
    u64 sum = 0;
    for (int j = tid; j < V; j += kThreads) {
      const float l = to_f32(row[j]);
      if (order_key(l) > f.key) sum += rule.weight(l);
    }
    sum = block_sum(sum, s_red) + (top_k - f.before) * rule.weight(key_logit(f.key));
    kept = min(kept, sum);
  }
  if (top_p > 0.0f && top_p < 1.0f) {
    const u64 target = part_of(top_p, whole);
    const Found f = reach<true>(row, V, rule, target, s_bins, s_pick);
    const u64 w = rule.weight(key_logit(f.key));
    kept = min(kept, f.before + (target - f.before + w - 1) / w * w);
  }
  const float uf = a.u[r];
  const u64 target = part_of(uf > 0.0f ? fminf(uf, 1.0f) : 0.0f, kept);
  const Found f = reach<true>(row, V, rule, target, s_bins, s_pick);
  const float l_at = key_logit(f.key);
  // among equal logits, the nth by index
  const u64 nth = (target - f.before + rule.weight(l_at) - 1) / rule.weight(l_at);
  u64 seen = 0;
  for (int j0 = 0; j0 < V; j0 += kThreads) {
    const int j = j0 + tid;
    const bool same = j < V && order_key(to_f32(row[j])) == f.key;
    const unsigned bal = __ballot_sync(0xffffffffu, same);
    __syncthreads();
    if (lane == 0) s_red[warp] = __popc(bal);
    __syncthreads();
    u64 mine = seen;
    for (int w = 0; w < warp; ++w) mine += s_red[w];
    mine += __popc(bal & ((1u << lane) - 1u)) + 1;
    if (same && mine == nth) {
      a.ids[r] = j;
      if (a.logprobs)
        a.logprobs[r] = static_cast<float>(log(rule.share(l_at) * rule.one / static_cast<double>(kept)));
    }
    for (int w = 0; w < 32; ++w) seen += s_red[w];
    if (seen >= nth) break;
  }
}

template <typename T>
cudaError_t launch(const LlmqSampleRows &a, cudaStream_t st) {
  int log2v = 0;
  while ((1 << log2v) < a.vocab) ++log2v;
  return serve_launch(k_sample_rows<T>, dim3(a.n_rows), dim3(kThreads), 0, st, a, 62 - log2v);
}

}  // namespace

extern "C" LLMQ_API int llmq_sample_rows(const LlmqSampleRows *a, void *stream) {
  ServeCheck c("llmq_sample_rows");
  c.require(a != nullptr, "null descriptor");
  if (c.rc != LLMQ_OK) return c.rc;
  c.require(serve_dtype(a->dtype), "unknown type of the logits");
  c.require(a->n_rows >= 0, "negative size");
  c.require(a->vocab > 0 && a->vocab <= (1 << 20), "vocab outside 1..2^20");
  if (c.rc != LLMQ_OK || a->n_rows == 0) return c.rc;
  c.require(a->logits && a->u && a->ids, "null pointer");
  c.require(a->stride >= a->vocab, "a row stride is shorter than its row");
  c.require(aligned_to(a->logits, serve_bytes(a->dtype)), "the logits do not start on an element");
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  c.launched(a->dtype == LLMQ_F32   ? launch<float>(*a, st)
             : a->dtype == LLMQ_F16 ? launch<__half>(*a, st)
                                    : launch<__nv_bfloat16>(*a, st));
  return c.rc;
}
