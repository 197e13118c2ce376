// llmq_paged.cu - the paged key-value cache on device memory: block tables and
// slot maps from request lengths (llmq_paged_plan), the cache's writer with
// RoPE (llmq_paged_append), and attention of one query row a sequence
// (llmq_paged_attention).
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "llmq_paged_attend.cuh"

using namespace llmq;

namespace {

// ==================================================================== plan
// Inclusive sum over the block's NT threads; *total receives the block's sum.
template <int NT>
__device__ __forceinline__ long long block_scan(long long v, long long *warp_sums, long long *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  long long w = lane < NT / 32 ? warp_sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < NT / 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  *total = __shfl_sync(0xffffffffu, w, NT / 32 - 1);
  const long long before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return v + (warp ? before : 0);
}

// Row r of request seq, whose rows end at row `end`.
__device__ __forceinline__ void plan_row(const LlmqPagedPlan &a, int r, int seq, int end, int len) {
  int pos = -1;
  long long slot = -1;
  if (seq >= 0) {
    pos = len - (end - r);
    const int at = pos / a.page_size, page = a.table[(long long)seq * a.table_stride + at];
    if (page >= 0)
      slot = (long long)page * a.page_size + (pos - at * a.page_size);
    else if (a.status)
      atomicOr(a.status, LLMQ_PAGED_BAD_PAGE);
  }
  a.slots[r] = slot;
  if (a.positions) a.positions[r] = pos;
  if (a.seqs) a.seqs[r] = seq;
  if (a.spans) a.spans[r] = pos + 1;
}

// What bounds a plan is latency: launches, the chain of sums and of each search (64 requests
// of one token 3.4 us; 1000 requests, 200 of them with prompts, some 100000 rows 10.8 us,
// of which their 2.5 MB would take 0.4).  So a small step is done by one CTA alone, rows
// and all; a larger one's rows take a second kernel (1000 requests with 1900 rows: 7.9 us
// in one, 8.1 us in two; 4800 rows: 11.0 and 9.0 us).
constexpr int kOneCtaRows = 2048;
// Up to this many requests and rows a CTA of 128 threads does, whose sums take fewer steps.
constexpr int kSmallSeqs = 128, kSmallRows = 512;

// One CTA: requests in chunks of NT, one a thread.  Sums in order: rows over the requests
// of valid lengths (which of them fit max_rows), pages over those (which fit the free
// pages), and, if a chunk refuses any, rows and pages over what is served (else those are
// the first two).  The chunk's new pages are then written by all threads, each finding its
// request by bisection of the page sums, and so are the rows of a small step.
template <int NT, bool rows_too>
__global__ void __launch_bounds__(NT) k_plan_scan(const LlmqPagedPlan a) {
  __shared__ long long s_warp[32];
  __shared__ long long s_end[NT];  // page sums up to and with each request
  __shared__ int s_have[NT], s_new[NT];
  __shared__ int s_row_end[rows_too ? NT : 1], s_len[rows_too ? NT : 1];
  serve_wait();
  serve_dependents();
  const int tid = threadIdx.x;
  const int given_head = a.free_head ? *a.free_head : 0;
  const bool bad_head = given_head < 0;
  const long long head = max(given_head, 0);
  const long long cap = (long long)a.max_pages * a.page_size;
  const int page_size = a.page_size;
  auto pages_of = [&](long long n) {  // n <= cap < 2^31
    return static_cast<int>((static_cast<uint32_t>(n) + static_cast<uint32_t>(page_size) - 1u) / static_cast<uint32_t>(page_size));
  };
  long long rows_seen = 0, pages_seen = 0, rows_done = 0, pages_done = 0;
  int flags = bad_head ? LLMQ_PAGED_NO_PAGES : 0;
  for (int b0 = 0; b0 < a.n_seqs; b0 += NT) {
    const int b = b0 + tid;
    const bool in = b < a.n_seqs;
    const long long cached = in ? a.cached[b] : 0, added = in ? a.added[b] : 0;
    const bool held = cached >= 0 && cached <= cap;
    const bool valid = held && added >= 0 && cached + added <= cap;
    if (in && !valid) flags |= LLMQ_PAGED_BAD_LEN;
    const int have = held ? pages_of(cached) : 0;
    long long chunk_rows, chunk_pages;
    const long long want = valid ? added : 0;
    const long long rows = block_scan<NT>(want, s_warp, &chunk_rows);
    const bool fits = valid && (want == 0 || rows_seen + rows <= a.max_rows);
    if (valid && !fits) flags |= LLMQ_PAGED_NO_ROWS;
    const int need = fits ? pages_of(cached + added) - have : 0;
    const long long pages = block_scan<NT>(need, s_warp, &chunk_pages);
    const bool served = fits && (need == 0 || (!bad_head && head + pages_seen + pages <= a.n_free));
    if (fits && !served) flags |= LLMQ_PAGED_NO_PAGES;
    rows_seen += chunk_rows;
    pages_seen += chunk_pages;
    const long long mine = served ? added : 0;
    const int fresh = served ? need : 0;
    long long row_sum = rows, page_sum = pages;
    if (__syncthreads_or(in && !served && want > 0)) {
      row_sum = block_scan<NT>(mine, s_warp, &chunk_rows);
      page_sum = block_scan<NT>(fresh, s_warp, &chunk_pages);
    }
    const long long end = rows_done + row_sum;
    const int len = held ? static_cast<int>(cached + mine) : 0;
    if (in) {
      a.first[b] = static_cast<int>(end - mine);
      a.lens[b] = len;
    }
    if (rows_too) {
      s_row_end[tid] = static_cast<int>(end);
      s_len[tid] = len;
    }
    s_end[tid] = page_sum;
    s_have[tid] = have;
    s_new[tid] = fresh;
    __syncthreads();
    for (long long j = tid; j < chunk_pages; j += NT) {
      int lo = 0, hi = NT - 1;  // the first request whose sum passes j
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > j)
          hi = mid;
        else
          lo = mid + 1;
      }
      const int at = s_have[lo] + static_cast<int>(j - (s_end[lo] - s_new[lo]));
      a.table[(long long)(b0 + lo) * a.table_stride + at] = a.free_pages[head + pages_done + j];
    }
    rows_done += chunk_rows;
    pages_done += chunk_pages;
    __syncthreads();
  }
  if (tid == 0) {
    a.first[a.n_seqs] = static_cast<int>(rows_done);
    if (a.next_head) *a.next_head = bad_head ? given_head : static_cast<int>(head + pages_done);
  }
  if (flags && a.status) atomicOr(a.status, flags);
  if (rows_too)
    for (int r = tid; r < a.max_rows; r += NT) {
      int lo = 0, hi = NT - 1;  // the first request whose rows end behind r
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_row_end[mid] > r)
          hi = mid;
        else
          lo = mid + 1;
      }
      const bool live = r < rows_done;
      plan_row(a, r, live ? lo : -1, live ? s_row_end[lo] : 0, live ? s_len[lo] : 0);
    }
}

constexpr int kFillThreads = 256;

// A thread a row, which finds its request by bisection of `first`.  A block brings it to
// shared memory first if it fits: one load's latency in place of one a step (the 1000
// requests above: 11.2 us without, 10.8 with).
constexpr int kFillSeqs = 4096;

__global__ void __launch_bounds__(kFillThreads) k_plan_fill(const LlmqPagedPlan a) {
  __shared__ int s_first[kFillSeqs + 1];
  serve_wait();
  serve_dependents();
  const int r = blockIdx.x * kFillThreads + threadIdx.x;
  const int *first = a.first;
  if (a.n_seqs <= kFillSeqs) {
    for (int i = threadIdx.x; i <= a.n_seqs; i += kFillThreads) s_first[i] = a.first[i];
    __syncthreads();
    first = s_first;
  }
  if (r >= a.max_rows) return;
  if (r >= first[a.n_seqs]) {
    plan_row(a, r, -1, 0, 0);
    return;
  }
  int lo = 0, hi = a.n_seqs - 1;  // the last request that starts at or before r
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  plan_row(a, r, lo, first[lo + 1], a.lens[lo]);
}

// ================================================================== append
struct AppendArgs {
  LlmqPagedKV kv;
  LlmqPagedAppend a;
};

constexpr int kAppendThreads = 256;
constexpr int kHeadLanes = 8;

// What bounds it: the rows' bytes, read once and written once.  16384 bf16 rows of 32 query
// heads and 8 KV heads of 128 (404 MB) take 70.9 us, 5.7 TB/s of the 6.46 a plain copy
// moves; 64 rows 4.1 us (3.3 from L2) and one 1.9 us, the latency of a launch and two
// dependent loads.
//
// A thread owns VN adjacent pairs (d, d + head_dim / 2) of every `lanes`th head of a row:
// the pairs' angles are read once and serve its heads.  The next head's loads are on
// their way before a head is stored (q_out may be q, so the compiler may not move a load
// over a store itself), the first head's before the row's slot is known.  Holding 2 to 6
// heads' loads at once took registers and so warps: 85 to 177 us for those rows.
template <typename T, typename KT, int VN>
__global__ void __launch_bounds__(kAppendThreads) k_append(const AppendArgs p, int chunks, int lanes) {
  serve_wait();
  serve_dependents();
  const LlmqPagedKV &kv = p.kv;
  const LlmqPagedAppend &a = p.a;
  const int per_row = chunks * lanes, rows_here = kAppendThreads / per_row;
  const int sub = threadIdx.x / per_row, t = threadIdx.x - sub * per_row;
  const int r = blockIdx.x * rows_here + sub;
  if (sub >= rows_here || r >= a.n_rows) return;
  const int hl = t / chunks, half = kv.head_dim / 2, d = (t - hl * chunks) * VN;
  const int nq = a.q ? a.n_heads : 0, heads = nq + 2 * kv.n_kv;
  const T *const qs = static_cast<const T *>(a.q) + r * a.q_stride + d;
  const T *const ks = static_cast<const T *>(a.k) + r * a.k_stride + d;
  const T *const vs = static_cast<const T *>(a.v) + r * a.v_stride + d;
  Pack<T, VN> x, y;
  auto load = [&](int h) {
    const T *src = h < nq              ? qs + (size_t)h * kv.head_dim
                   : h < nq + kv.n_kv ? ks + (size_t)(h - nq) * kv.head_dim
                                        : vs + (size_t)(h - nq - kv.n_kv) * kv.head_dim;
    x = *reinterpret_cast<const Pack<T, VN> *>(src);
    y = *reinterpret_cast<const Pack<T, VN> *>(src + half);
  };
  if (hl < heads) load(hl);
  const long long slot = a.slots[r];
  const bool turn = a.rope_cos != nullptr;
  const int pos = turn ? a.positions[r] : 0;
  if (slot < 0) return;
  if (slot >= (long long)kv.n_pages * kv.page_size) {
    if (t == 0 && a.status) atomicOr(a.status, LLMQ_PAGED_BAD_SLOT);
    return;
  }
  if (turn && (pos < 0 || pos >= a.rope_len)) {
    if (t == 0 && a.status) atomicOr(a.status, LLMQ_PAGED_BAD_POS);
    return;
  }
  Pack<float, VN> cs, sn;
  if (turn) {
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      cs.v[i] = a.rope_cos[(size_t)pos * half + d + i];
      sn.v[i] = a.rope_sin[(size_t)pos * half + d + i];
    }
  }
  const int page = static_cast<int>(slot) / kv.page_size, token = static_cast<int>(slot) - page * kv.page_size;
  const long long at = page * kv.page_stride + token * kv.token_stride;
  for (int h = hl; h < heads; h += lanes) {
    const bool is_q = h < nq, is_k = !is_q && h < nq + kv.n_kv;
    const int hh = is_q ? h : is_k ? h - nq : h - nq - kv.n_kv;
    const Pack<T, VN> x0 = x, y0 = y;
    if (h + lanes < heads) load(h + lanes);
    auto put = [&](auto *dst) {
      using D = std::remove_pointer_t<decltype(dst)>;
      Pack<D, VN> lo, hi;
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        float u = to_f32(x0.v[i]), w = to_f32(y0.v[i]);
        if (turn && (is_q || is_k)) {  // rope.c:58-64, the products rounded on their own
          const float a0 = u, b0 = w;
          u = __fsub_rn(__fmul_rn(a0, cs.v[i]), __fmul_rn(b0, sn.v[i]));
          w = __fadd_rn(__fmul_rn(b0, cs.v[i]), __fmul_rn(a0, sn.v[i]));
        }
        lo.v[i] = from_f32<D>(u);
        hi.v[i] = from_f32<D>(w);
      }
      *reinterpret_cast<Pack<D, VN> *>(dst) = lo;
      *reinterpret_cast<Pack<D, VN> *>(dst + half) = hi;
    };
    if (is_q)
      put(static_cast<T *>(a.q_out) + r * a.q_out_stride + (size_t)hh * kv.head_dim + d);
    else
      put(static_cast<KT *>(is_k ? kv.k : kv.v) + at + hh * kv.head_stride + d);
  }
}

// ------------------------------------------------------------- host checks
void check_pool(ServeCheck &c, const LlmqPagedKV *kv) {
  c.require(kv != nullptr, "null pool");
  if (c.rc != LLMQ_OK) return;
  c.require(kv->k && kv->v, "null pool memory");
  c.require(serve_dtype(kv->dtype), "unknown type of the pool");
  c.require(kv->n_pages > 0 && kv->page_size > 0 && (long long)kv->n_pages * kv->page_size <= INT_MAX,
            "the pool needs n_pages > 0, page_size > 0 and fewer than 2^31 slots");
  c.require(kv->n_kv > 0 && kv->n_kv <= 65535, "n_kv outside 1..65535");
  c.require(kv->head_dim > 0 && kv->head_dim <= 256 && kv->head_dim % 8 == 0,
            "head_dim must be a multiple of 8, at most 256");
  if (c.rc != LLMQ_OK) return;
  const long long e = static_cast<long long>(serve_bytes(kv->dtype));
  c.require(aligned16(kv->k) && aligned16(kv->v), "pool memory must start on 16 bytes");
  c.require(kv->page_stride >= 0 && kv->token_stride >= 0 && kv->head_stride >= 0 && kv->page_stride * e % 16 == 0 &&
                kv->token_stride * e % 16 == 0 && kv->head_stride * e % 16 == 0,
            "pool strides must be multiples of 16 bytes, none negative");
}

}  // namespace

extern "C" LLMQ_API int llmq_paged_plan(const LlmqPagedPlan *a, void *stream) {
  ServeCheck c("llmq_paged_plan");
  c.require(a != nullptr, "null descriptor");
  if (c.rc != LLMQ_OK) return c.rc;
  c.require(a->n_seqs >= 0 && a->max_rows >= 0 && a->n_free >= 0, "negative size");
  c.require(a->n_seqs <= kServeMaxRows, "n_seqs is above 2^31 - 4097");
  c.require(a->page_size > 0 && a->max_pages > 0 && (long long)a->page_size * a->max_pages <= INT_MAX,
            "page_size and max_pages must be above 0 and their product below 2^31");
  c.require(a->table_stride >= a->max_pages, "table_stride is below max_pages");
  c.require(a->n_seqs == 0 || (a->cached && a->added && a->table && a->lens), "null pointer");
  c.require(a->first && (a->max_rows == 0 || a->slots) && (a->n_free == 0 || a->free_pages), "null pointer");
  c.elements(a->cached, "cached");
  c.elements(a->added, "added");
  c.elements(a->free_pages, "free_pages");
  c.elements(a->free_head, "free_head");
  c.elements(a->table, "table");
  c.elements(a->lens, "lens");
  c.elements(a->first, "first");
  c.elements(a->slots, "slots");
  c.elements(a->positions, "positions");
  c.elements(a->seqs, "seqs");
  c.elements(a->spans, "spans");
  c.elements(a->next_head, "next_head");
  c.elements(a->status, "status");
  c.on_device();
  c.memory(a->cached, "cached");
  c.memory(a->added, "added");
  c.memory(a->free_pages, "free_pages");
  c.memory(a->free_head, "free_head");
  c.memory(a->table, "table");
  c.memory(a->lens, "lens");
  c.memory(a->first, "first");
  c.memory(a->slots, "slots");
  c.memory(a->positions, "positions");
  c.memory(a->seqs, "seqs");
  c.memory(a->spans, "spans");
  c.memory(a->next_head, "next_head");
  c.memory(a->status, "status");
  if (c.rc != LLMQ_OK) return c.rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool one = a->n_seqs <= 1024 && a->max_rows <= kOneCtaRows;
  if (a->n_seqs <= kSmallSeqs && a->max_rows <= kSmallRows)
    c.launched(serve_launch(k_plan_scan<128, true>, dim3(1), dim3(128), 0, st, *a));
  else
    c.launched(serve_launch(one ? k_plan_scan<1024, true> : k_plan_scan<1024, false>, dim3(1), dim3(1024), 0, st, *a));
  if (c.rc == LLMQ_OK && !one && a->max_rows > 0)
    c.launched(serve_launch(k_plan_fill, dim3((a->max_rows - 1) / kFillThreads + 1), dim3(kFillThreads), 0, st, *a));
  return c.rc;
}

namespace {

template <typename T, typename KT>
cudaError_t launch_append(const AppendArgs &p, cudaStream_t st) {
  const LlmqPagedAppend &a = p.a;
  constexpr int kWide = 16 / sizeof(T);
  const int half = p.kv.head_dim / 2;
  auto wide = [&](const void *x, long long stride) {
    return !x || (aligned16(x) && stride * (long long)sizeof(T) % 16 == 0);
  };
  const bool vec = half % kWide == 0 && wide(a.q, a.q_stride) && wide(a.k, a.k_stride) && wide(a.v, a.v_stride) &&
                   wide(a.q_out, a.q_out_stride);
  const int chunks = vec ? half / kWide : half;
  const int lanes = std::min(kHeadLanes, kAppendThreads / chunks), rows_here = kAppendThreads / (chunks * lanes);
  const dim3 grid((a.n_rows - 1) / rows_here + 1);
  return vec ? serve_launch(k_append<T, KT, kWide>, grid, dim3(kAppendThreads), 0, st, p, chunks, lanes)
             : serve_launch(k_append<T, KT, 1>, grid, dim3(kAppendThreads), 0, st, p, chunks, lanes);
}

template <typename Core, int HDP>
cudaError_t launch_attend(AttendArgs p, int sms, cudaStream_t st) {
  typedef AttendShape<Core, HDP> Sh;
  const LlmqPagedAttention &a = p.a;
  const int group = a.n_heads / p.kv.n_kv, total_rows = a.n_rows;
  p.blocks = (group + Core::kBlock - 1) / Core::kBlock;
  cudaError_t e = cudaFuncSetAttribute(k_attend<Core, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
  for (p.row0 = 0; p.row0 < total_rows && e == cudaSuccess; p.row0 += kAttendMaxRows) {
    p.rows = std::min(kAttendMaxRows, total_rows - p.row0);
    // no more CTAs than tiles there can be
    const long long tiles = (long long)p.rows * p.kv.n_kv * p.blocks *
                            (((long long)a.max_pages * p.kv.page_size + Sh::kTile - 1) / Sh::kTile);
    const int ctas = static_cast<int>(
        std::max(1LL, std::min<long long>({tiles, (long long)sms * Sh::kPerSm, (long long)kAttendMaxCtas})));
    e = serve_launch(k_attend<Core, HDP>, dim3(ctas), dim3(kAttendThreads), Sh::kSmem, st, p);
    if (e == cudaSuccess && ctas > 1)
      e = serve_launch(k_attend_join<typename Core::Row>, dim3(ctas, std::min(group, (int)Core::kBlock)),
                       dim3(kJoinThreads), 0, st, p, ctas, (int)Core::kBlock);
  }
  return e;
}

template <typename T, typename KT>
cudaError_t attend_by_shape(const AttendArgs &p, int sms, cudaStream_t st) {
  const int hd = p.kv.head_dim;
  if constexpr (std::is_same<KT, float>::value) {
    const int group = p.a.n_heads / p.kv.n_kv;
    if (group <= 4) {
      if (hd <= 64) return launch_attend<CoreF32<64, 4>, 64>(p, sms, st);
      if (hd <= 128) return launch_attend<CoreF32<128, 4>, 128>(p, sms, st);
      return launch_attend<CoreF32<256, 4>, 256>(p, sms, st);
    }
    if (hd <= 64) return launch_attend<CoreF32<64, 8>, 64>(p, sms, st);
    if (hd <= 128) return launch_attend<CoreF32<128, 8>, 128>(p, sms, st);
    return launch_attend<CoreF32<256, 8>, 256>(p, sms, st);
  } else {
    if (hd <= 64) return launch_attend<CoreMma<T, KT, 64>, 64>(p, sms, st);
    if (hd <= 96) return launch_attend<CoreMma<T, KT, 96>, 96>(p, sms, st);
    if (hd <= 128) return launch_attend<CoreMma<T, KT, 128>, 128>(p, sms, st);
    return launch_attend<CoreMma<T, KT, 256>, 256>(p, sms, st);
  }
}

// f(T, KT) for a type of the rows and one of the pool that check_types let through.
template <typename F>
cudaError_t by_types(int t, int kt, F f) {
  if (t == LLMQ_F16) return f(__half(), __half());
  if (t == LLMQ_BF16) return f(__nv_bfloat16(), __nv_bfloat16());
  if (kt == LLMQ_F16) return f(float(), __half());
  if (kt == LLMQ_BF16) return f(float(), __nv_bfloat16());
  return f(float(), float());
}

void check_types(ServeCheck &c, int t, int kt) {
  c.require(serve_dtype(t), "unknown type of the rows");
  c.require(t == kt || t == LLMQ_F32, "the rows must have the pool's type or be f32");
}

}  // namespace

extern "C" LLMQ_API int llmq_paged_append(const LlmqPagedKV *kv, const LlmqPagedAppend *a, void *stream) {
  ServeCheck c("llmq_paged_append");
  c.require(a != nullptr, "null descriptor");
  check_pool(c, kv);
  if (c.rc != LLMQ_OK) return c.rc;
  check_types(c, a->dtype, kv->dtype);
  c.require(a->n_rows >= 0 && a->n_heads >= 0 && a->rope_len >= 0, "negative size");
  c.require(a->n_rows <= kServeMaxRows, "n_rows is above 2^31 - 4097");
  c.require((long long)a->n_heads * kv->head_dim <= INT_MAX, "a row has 2^31 elements or more");
  if (c.rc != LLMQ_OK || a->n_rows == 0) return c.rc;
  c.require(a->k && a->v && a->slots, "null pointer");
  c.require((a->n_heads > 0) == (a->q != nullptr) && (a->q != nullptr) == (a->q_out != nullptr),
            "q, q_out and n_heads go together");
  c.require((a->rope_cos != nullptr) == (a->rope_sin != nullptr), "one angle table without the other");
  c.require(!a->rope_cos || (a->positions && a->rope_len > 0), "angle tables without positions or rope_len");
  const long long kvd = (long long)kv->n_kv * kv->head_dim, qd = (long long)a->n_heads * kv->head_dim;
  c.require(a->k_stride >= kvd && a->v_stride >= kvd && a->q_stride >= (a->q ? qd : 0) &&
                a->q_out_stride >= (a->q ? qd : 0),
            "a row stride is shorter than its row");
  const size_t e = c.rc == LLMQ_OK ? serve_bytes(a->dtype) : 1;
  c.require(aligned_to(a->q, e) && aligned_to(a->k, e) && aligned_to(a->v, e) && aligned_to(a->q_out, e),
            "a row does not start on an element");
  c.elements(a->slots, "slots");
  c.elements(a->positions, "positions");
  c.elements(a->rope_cos, "rope_cos");
  c.elements(a->rope_sin, "rope_sin");
  c.elements(a->status, "status");
  c.on_device();
  c.memory(kv->k, "the pool");
  c.memory(kv->v, "the pool");
  c.memory(a->q, "q");
  c.memory(a->k, "k");
  c.memory(a->v, "v");
  c.memory(a->q_out, "q_out");
  c.memory(a->slots, "slots");
  c.memory(a->positions, "positions");
  c.memory(a->rope_cos, "rope_cos");
  c.memory(a->rope_sin, "rope_sin");
  c.memory(a->status, "status");
  if (c.rc != LLMQ_OK) return c.rc;
  const AppendArgs p{*kv, *a};
  c.launched(by_types(a->dtype, kv->dtype, [&](auto t, auto kt) {
    return launch_append<decltype(t), decltype(kt)>(p, static_cast<cudaStream_t>(stream));
  }));
  return c.rc;
}

extern "C" LLMQ_API size_t llmq_paged_attention_workspace(int n_rows, int n_heads, int n_kv, int head_dim) {
  if (n_rows < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv != 0 || head_dim <= 0 || head_dim > 256 ||
      head_dim % 8 != 0) {
    llmq_set_error(LLMQ_ERR_ARG, "llmq_paged_attention_workspace: bad sizes (%d rows, %d / %d heads of %d)", n_rows,
                   n_heads, n_kv, head_dim);
    return 0;
  }
  return attend_workspace(head_dim);
}

extern "C" LLMQ_API int llmq_paged_attention(const LlmqPagedKV *kv, const LlmqPagedAttention *a, void *stream) {
  ServeCheck c("llmq_paged_attention");
  c.require(a != nullptr, "null descriptor");
  check_pool(c, kv);
  if (c.rc != LLMQ_OK) return c.rc;
  check_types(c, a->dtype, kv->dtype);
  c.require(a->n_rows >= 0 && a->n_seqs >= 0 && a->max_pages >= 0 && a->window >= 0, "negative size");
  c.require(a->n_rows <= kServeMaxRows, "n_rows is above 2^31 - 4097");
  c.require(a->n_heads > 0 && a->n_heads % kv->n_kv == 0, "n_heads must be a multiple of n_kv");
  c.require((long long)a->n_heads * kv->head_dim <= INT_MAX, "a row has 2^31 elements or more");
  // (a tile may reach past the last position: room for it below 2^31)
  c.require((long long)a->max_pages * kv->page_size <= INT_MAX - 4096, "max_pages * page_size must stay below 2^31 - 4096");
  c.require(a->table_stride >= a->max_pages, "table_stride is below max_pages");
  c.require(std::isfinite(a->scale), "scale is not finite");
  if (c.rc != LLMQ_OK || a->n_rows == 0) return c.rc;
  c.require(a->q && a->out && a->lens && (a->table || a->max_pages == 0 || a->n_seqs == 0), "null pointer");
  c.require(a->seqs || a->n_seqs >= a->n_rows, "n_seqs is below n_rows and seqs is null");
  const long long qd = (long long)a->n_heads * kv->head_dim;
  c.require(a->q_stride >= qd && a->out_stride >= qd, "a row stride is shorter than its row");
  const size_t e = c.rc == LLMQ_OK ? serve_bytes(a->dtype) : 1;
  c.require(aligned_to(a->q, e) && aligned_to(a->out, e), "a row does not start on an element");
  c.elements(a->lse, "lse");
  c.elements(a->table, "table");
  c.elements(a->seqs, "seqs");
  c.elements(a->lens, "lens");
  c.elements(a->status, "status");
  if (c.rc != LLMQ_OK) return c.rc;
  const size_t need = llmq_paged_attention_workspace(a->n_rows, a->n_heads, kv->n_kv, kv->head_dim);
  c.require(a->workspace && a->workspace_bytes >= need && aligned16(a->workspace),
            "the workspace is missing, too small or not on 16 bytes");
  c.on_device();
  c.memory(kv->k, "the pool");
  c.memory(kv->v, "the pool");
  c.memory(a->q, "q");
  c.memory(a->out, "out");
  c.memory(a->lse, "lse");
  c.memory(a->table, "table");
  c.memory(a->seqs, "seqs");
  c.memory(a->lens, "lens");
  c.memory(a->workspace, "workspace");
  c.memory(a->status, "status");
  if (c.rc != LLMQ_OK) return c.rc;
  AttendArgs p{};
  p.kv = *kv;
  p.a = *a;
  p.scale_log2 = (a->scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(kv->head_dim)) : a->scale) * 1.44269504088896341f;
  const long long e_pool = static_cast<long long>(serve_bytes(kv->dtype));
  p.page_bytes = kv->page_stride * e_pool;
  p.token_bytes = kv->token_stride * e_pool;
  p.head_bytes = kv->head_stride * e_pool;
  set_division(p);
  int sms = 0;
  c.launched(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c.device));
  if (c.rc != LLMQ_OK) return c.rc;
  c.launched(by_types(a->dtype, kv->dtype, [&](auto t, auto kt) {
    return attend_by_shape<decltype(t), decltype(kt)>(p, sms, static_cast<cudaStream_t>(stream));
  }));
  return c.rc;
}
