// llmq_paged_model.cuh - a model's batches over a paged cache (q_llama_paged_*) and
// sampled batched decode.  The part of llmq_dev.cu that joins its multi-row pass with
// the serving operators; included at that file's end.
#pragma once

// Pools of all layers, the sequences' tables, and what one step of the batch needs.
// The GPU holds the tables, lengths and free pages, which llmq_paged_plan advances;
// the host mirrors the lengths and each sequence's pages, so that a step that cannot
// be served is refused before anything runs.
struct LlmqPagedCache {
  DevModel *model = nullptr;
  int n_pages = 0, page_size = 0, max_seqs = 0, max_pages = 0, dtype = 0;
  bool broken = false;
  char *k = nullptr, *v = nullptr;  // [layer][page][position][head][head_dim]
  int *table = nullptr, *lens = nullptr, *first = nullptr, *added = nullptr, *free_pages = nullptr, *head = nullptr;
  int *status = nullptr, *last = nullptr;  // last: the rows the lm-head takes
  int *h_step = nullptr;                   // pinned: added [max_seqs], then last [max_seqs]
  float *x = nullptr;                      // [max_seqs][d_model]: their residual stream
  void *work = nullptr;
  size_t work_bytes = 0;
  // of a step's rows
  int cap = 0;
  long long *slots = nullptr;
  int *positions = nullptr, *seqs = nullptr, *spans = nullptr;
  // host mirror
  std::vector<std::vector<int>> pages;
  std::vector<int> len, free_list;  // free_list[head_h ..] as on the GPU
  int head_h = 0;
  size_t layer_bytes() const {
    return (size_t)n_pages * page_size * model->kvd * (dtype == LLMQ_F32 ? 4 : 2);
  }
};

namespace {

void release_paged(LlmqPagedCache *c) {
  void *p[] = {c->k,      c->v,    c->table, c->lens,      c->first, c->added, c->free_pages, c->head, c->status,
               c->last,   c->x,    c->work,  c->slots,     c->positions, c->seqs, c->spans};
  for (void *q : p) cudaFree(q);
  cudaFreeHost(c->h_step);
  delete c;
}

// The cache behind a handle, with its model's GPU current if `select`; null if it is none.
LlmqPagedCache *find_paged(const LlmqPagedCache *handle, const char *fn, bool select) {
  for (auto &m : g_models)
    for (LlmqPagedCache *c : m.second->paged)
      if (c == handle) {
        if (!select || cudaSetDevice(c->model->device) == cudaSuccess) return c;
        llmq_set_error(LLMQ_ERR_CUDA, "%s: cannot select device %d", fn, c->model->device);
        return nullptr;
      }
  llmq_set_error(LLMQ_ERR_STATE, "%s: not a paged cache of a loaded model", fn);
  return nullptr;
}

int paged_attention(const LlmqPagedCache &c, DevModel *M, int layer, int row0, int rows) {
  const LlmqConfig &cfg = M->cfg;
  const int hd = cfg.head_dim, qd = M->qd, kvd = M->kvd;
  auto &R = M->rows;
  LlmqPagedKV kv{};
  kv.k = c.k + layer * c.layer_bytes();
  kv.v = c.v + layer * c.layer_bytes();
  kv.dtype = c.dtype;
  kv.n_pages = c.n_pages;
  kv.page_size = c.page_size;
  kv.n_kv = cfg.n_kv;
  kv.head_dim = hd;
  kv.head_stride = hd;
  kv.token_stride = kvd;
  kv.page_stride = (long long)c.page_size * kvd;
  LlmqPagedAppend ap{};
  ap.n_rows = rows;
  ap.n_heads = cfg.n_heads;
  ap.dtype = LLMQ_F32;
  ap.rope_len = cfg.max_seq;
  ap.q = R.qkv;
  ap.k = R.qkv + qd;
  ap.v = R.qkv + qd + kvd;
  ap.q_stride = ap.k_stride = ap.v_stride = qd + 2 * kvd;
  ap.q_out = R.qr;
  ap.q_out_stride = qd;
  ap.slots = c.slots + row0;
  ap.positions = c.positions + row0;
  ap.rope_cos = M->rope_cos;
  ap.rope_sin = M->rope_sin;
  ap.status = c.status;
  LlmqPagedAttention at{};
  at.n_rows = rows;
  at.n_heads = cfg.n_heads;
  at.dtype = LLMQ_F32;
  at.max_pages = c.max_pages;
  at.n_seqs = c.max_seqs;
  at.q = R.qr;
  at.q_stride = qd;
  at.out = R.ao;
  at.out_stride = qd;
  at.table = c.table;
  at.table_stride = c.max_pages;
  at.seqs = c.seqs + row0;
  at.lens = c.spans + row0;
  at.workspace = c.work;
  at.workspace_bytes = c.work_bytes;
  at.status = c.status;
  return llmq_paged_append(&kv, &ap, M->stream) == LLMQ_OK && llmq_paged_attention(&kv, &at, M->stream) == LLMQ_OK;
}

// Rows last[i] of a pass over rows [row0, row0 + rows) to x_out[i].
__global__ void __launch_bounds__(256) k_take_rows(const float *x, const int *last, int row0, int rows, int dm,
                                                   float *x_out) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = last[blockIdx.x] - row0;
  if (r < 0 || r >= rows) return;
  for (int d = threadIdx.x; d < dm; d += 256) x_out[(size_t)blockIdx.x * dm + d] = x[(size_t)r * dm + d];
}

LlmqPagedCache *paged_create(const QLlamaModel *m, int n_pages, int page_size, int max_seqs, int dtype) {
  const char *fn = "q_llama_paged_create";
  // (llmq_paged_attention's limit on a table row, so that no step is refused half way)
  if (n_pages <= 0 || page_size <= 0 || max_seqs <= 0 || (long long)n_pages * page_size > INT_MAX - 4096 ||
      dtype < LLMQ_F32 || dtype > LLMQ_BF16) {
    llmq_set_error(LLMQ_ERR_ARG, "%s: bad sizes or type (%d pages of %d, %d sequences)", fn, n_pages, page_size,
                   max_seqs);
    return nullptr;
  }
  if (g_tp.world > 1) {
    llmq_set_error(LLMQ_ERR_STATE, "%s: not under tensor parallelism", fn);
    return nullptr;
  }
  if (m && (m->head_dim <= 0 || m->head_dim % 8 != 0 || m->head_dim > 256)) {
    llmq_set_error(LLMQ_ERR_ARG, "%s: head_dim %d is not a multiple of 8 up to 256", fn, m->head_dim);
    return nullptr;
  }
  DevModel *M = get_model(m);
  if (!M) return nullptr;
  const LlmqConfig &cfg = M->cfg;
  LlmqPagedCache *c = new LlmqPagedCache();
  c->model = M;
  c->n_pages = n_pages;
  c->page_size = page_size;
  c->max_seqs = max_seqs;
  c->max_pages = static_cast<int>(std::min<long long>(n_pages, ((long long)cfg.max_seq + page_size - 1) / page_size));
  c->dtype = dtype;
  try {
    c->pages.resize((size_t)max_seqs);
    c->len.assign((size_t)max_seqs, 0);
    c->free_list.resize((size_t)n_pages);
  } catch (...) {
    release_paged(c);
    throw;
  }
  for (int i = 0; i < n_pages; ++i) c->free_list[i] = i;
  c->work_bytes = llmq_paged_attention_workspace(1, cfg.n_heads, cfg.n_kv, cfg.head_dim);
  const size_t pool = c->layer_bytes() * cfg.n_layers;
  auto ok = [&]() -> int {
    CK(cudaMalloc(&c->k, pool));
    CK(cudaMalloc(&c->v, pool));
    CK(cudaMalloc(&c->work, c->work_bytes));
    CK(cudaMalloc(&c->table, (size_t)max_seqs * c->max_pages * sizeof(int)));
    CK(cudaMallocHost(&c->h_step, 2 * (size_t)max_seqs * sizeof(int)));
    CK(cudaMalloc(&c->x, (size_t)max_seqs * cfg.d_model * sizeof(float)));
    if (!dev_zeros(&c->lens, max_seqs) || !dev_zeros(&c->first, (size_t)max_seqs + 1) || !dev_zeros(&c->added, max_seqs) ||
        !dev_zeros(&c->head, 1) || !dev_zeros(&c->status, 1) || !dev_zeros(&c->last, max_seqs) ||
        !dev_upload(&c->free_pages, c->free_list.data(), c->free_list.size()))
      return 0;
    CK(cudaMemset(c->table, 0xff, (size_t)max_seqs * c->max_pages * sizeof(int)));
    CK(cudaStreamSynchronize(nullptr));
    return 1;
  };
  if (!ok()) {
    release_paged(c);
    return nullptr;
  }
  try {
    M->paged.push_back(c);
  } catch (...) {
    release_paged(c);
    throw;
  }
  return c;
}

int paged_reset(LlmqPagedCache *c, int seq) {
  const cudaStream_t st = c->model->stream;
  std::vector<int> &own = c->pages[(size_t)seq];
  std::vector<int> next;
  if (!own.empty()) {
    next.assign(c->free_list.begin() + c->head_h, c->free_list.end());
    next.insert(next.end(), own.begin(), own.end());
  }
  c->broken = true;  // a failure from here on leaves the GPU's lists behind the host's
  if (!own.empty()) {
    CK(cudaMemcpyAsync(c->free_pages, next.data(), next.size() * sizeof(int), cudaMemcpyHostToDevice, st));
    CK(cudaMemsetAsync(c->head, 0, sizeof(int), st));
  }
  CK(cudaMemsetAsync(c->lens + seq, 0, sizeof(int), st));
  CK(cudaStreamSynchronize(st));  // `next` has been read
  if (!own.empty()) {
    c->free_list.swap(next);
    c->head_h = 0;
    own.clear();
  }
  c->len[(size_t)seq] = 0;
  c->broken = false;
  return 1;
}

// Everything a step of T rows, n_active of them for the lm-head, would allocate on its way.
int paged_reserve(DevCtx &ctx, DevModel *M, int T, int n_active) {
  const LlmqConfig &cfg = M->cfg;
  TcArgs t;
  // a full pass, if there is one, and the last
  for (int rows : {std::min(T, kRowsPerPass), T % kRowsPerPass}) {
    if (rows == 0) continue;
    if (!ensure_pass(ctx, M, rows, 0, false)) return 0;
    for (int l = 0; l < cfg.n_layers; ++l)
      for (const Mat *w : {&M->qkv[l], &M->wo[l], &M->w13[l], &M->w2[l]})
        if (!plan_tc(ctx, *w, rows, t)) return 0;
  }
  for (int rows : {std::min(n_active, kRowsPerPass), n_active % kRowsPerPass})
    if (rows > 0 && (!ensure_pass(ctx, M, rows, rows, false) || !plan_tc(ctx, M->lm, rows, t))) return 0;
  return 1;
}

int paged_step(const QLlamaModel *m, LlmqPagedCache *c, const int *added, const int *tokens, const LlmqSampling *s,
               int *ids, Tensor *logits) {
  const char *fn = "q_llama_paged_step";
  if (!added || !ids || (s && !s->u)) {
    llmq_set_error(LLMQ_ERR_ARG, "%s: null pointer", fn);
    return 0;
  }
  DevModel *M = get_model(m);
  if (!M) return 0;
  if (c->model != M) {
    llmq_set_error(LLMQ_ERR_STATE, "%s: this cache belongs to another model", fn);
    return 0;
  }
  if (c->broken || g_tp.world > 1) {
    llmq_set_error(LLMQ_ERR_STATE, "%s: %s", fn, c->broken ? "an earlier step failed on the GPU" : "not under tensor parallelism");
    return 0;
  }
  DevCtx *ctx = get_ctx();
  if (!ctx) return 0;
  const LlmqConfig &cfg = M->cfg;
  const long long cap = std::min<long long>(cfg.max_seq, (long long)c->max_pages * c->page_size);
  // ---- can it be served?
  long long total = 0;
  std::vector<int> active, last;
  std::vector<int> need((size_t)c->max_seqs, 0);
  long long new_pages = 0;
  for (int b = 0; b < c->max_seqs; ++b) {
    if (added[b] < 0 || c->len[b] + (long long)added[b] > cap) {
      llmq_set_error(LLMQ_ERR_ARG, "%s: sequence %d: %d + %d positions exceed %lld", fn, b, c->len[b], added[b], cap);
      return 0;
    }
    if (added[b] == 0) continue;
    total += added[b];
    if (total > INT_MAX / 2) {
      llmq_set_error(LLMQ_ERR_ARG, "%s: too many tokens", fn);
      return 0;
    }
    active.push_back(b);
    last.push_back(static_cast<int>(total) - 1);
    need[b] = (c->len[b] + added[b] + c->page_size - 1) / c->page_size - static_cast<int>(c->pages[b].size());
    new_pages += need[b];
  }
  for (int b = 0; b < c->max_seqs; ++b) ids[b] = -1;
  if (active.empty()) return 1;
  const int T = static_cast<int>(total), n_active = static_cast<int>(active.size());
  if (new_pages > (long long)c->free_list.size() - c->head_h) {
    llmq_set_error(LLMQ_ERR_OOM, "%s: %lld pages needed, %lld free", fn, new_pages,
                   (long long)c->free_list.size() - c->head_h);
    return 0;
  }
  if (!tokens || (logits && (!logits->data || logits->size < (size_t)n_active * cfg.vocab))) {
    llmq_set_error(LLMQ_ERR_ARG, "%s: null tokens, or a logits tensor below %d x %d floats", fn, n_active, cfg.vocab);
    return 0;
  }
  std::vector<RowDesc> rows((size_t)T);
  for (int r = 0; r < T; ++r) {
    if (tokens[r] < 0 || tokens[r] >= cfg.vocab) {
      llmq_set_error(LLMQ_ERR_ARG, "%s: token id %d at %d outside [0, %d)", fn, tokens[r], r, cfg.vocab);
      return 0;
    }
    rows[r] = RowDesc{nullptr, nullptr, 0, 0, tokens[r], 0};
  }
  for (int b : active) {  // room for the pages it takes, so that noting them cannot fail
    std::vector<int> &own = c->pages[b];
    const size_t n = own.size() + need[b];
    if (n > own.capacity()) own.reserve(std::max(n, 2 * own.capacity()));
  }
  if (T > c->cap) {
    void *old[] = {c->slots, c->positions, c->seqs, c->spans};
    for (void *p : old) cudaFree(p);
    c->slots = nullptr;
    c->positions = c->seqs = c->spans = nullptr;
    c->cap = 0;
    CK(cudaMalloc(&c->slots, (size_t)T * sizeof(long long)));
    CK(cudaMalloc(&c->positions, (size_t)T * sizeof(int)));
    CK(cudaMalloc(&c->seqs, (size_t)T * sizeof(int)));
    CK(cudaMalloc(&c->spans, (size_t)T * sizeof(int)));
    c->cap = T;
  }
  LlmqSampleRows limits{};
  limits.vocab = cfg.vocab;
  limits.dtype = LLMQ_F32;
  if (s && llmq_sample_rows(&limits, M->stream) != LLMQ_OK) return 0;  // (no rows: its checks alone)
  if (!paged_reserve(*ctx, M, T, n_active)) return 0;
  std::vector<int> drawn((size_t)n_active);
  SampleColumns cols;
  if (s && !cols.fill(M, *s, n_active, active.data())) return 0;
  // ---- from here on a failure leaves the GPU's tables behind the host's
  c->broken = true;
  std::copy(added, added + c->max_seqs, c->h_step);
  std::copy(last.begin(), last.end(), c->h_step + c->max_seqs);
  CK(cudaMemcpyAsync(c->added, c->h_step, (size_t)c->max_seqs * sizeof(int), cudaMemcpyHostToDevice, M->stream));
  CK(cudaMemcpyAsync(c->last, c->h_step + c->max_seqs, last.size() * sizeof(int), cudaMemcpyHostToDevice, M->stream));
  g_launches = 0;
  const long long served = t_serve_launches;
  CK(cudaEventRecord(M->ev0, M->stream));
  LlmqPagedPlan plan{};
  plan.n_seqs = c->max_seqs;
  plan.page_size = c->page_size;
  plan.max_pages = c->max_pages;
  plan.max_rows = T;
  plan.n_free = static_cast<int>(c->free_list.size());
  plan.cached = c->lens;
  plan.added = c->added;
  plan.free_pages = c->free_pages;
  plan.free_head = plan.next_head = c->head;
  plan.table = c->table;
  plan.table_stride = c->max_pages;
  plan.lens = c->lens;
  plan.first = c->first;
  plan.slots = c->slots;
  plan.positions = c->positions;
  plan.seqs = c->seqs;
  plan.spans = c->spans;
  plan.status = c->status;
  if (llmq_paged_plan(&plan, M->stream) != LLMQ_OK) return 0;
  for (int off = 0; off < T; off += kRowsPerPass) {
    const int n = std::min(kRowsPerPass, T - off);
    RowsHook hook;
    hook.paged = c;
    hook.row0 = off;
    if (!run_rows(*ctx, M, rows.data() + off, n, n, nullptr, nullptr, hook)) return 0;
    CK(launch_pdl(k_take_rows, dim3(n_active), dim3(256), 0, M->stream, static_cast<const float *>(M->rows.x),
                  static_cast<const int *>(c->last), off, n, cfg.d_model, c->x));
  }
  for (int off = 0; off < n_active; off += kRowsPerPass) {
    const int n = std::min(kRowsPerPass, n_active - off);
    RowsHook hook;
    LlmqSampleRows sr{};
    hook.x = c->x + (size_t)off * cfg.d_model;
    if (s) {
      sr = cols.rows(off);
      hook.sample = &sr;
    }
    if (!run_rows(*ctx, M, rows.data(), n, 0, logits ? logits->data + (size_t)off * cfg.vocab : nullptr,
                  drawn.data() + off, hook))
      return 0;
  }
  int flags = 0;
  CK(cudaMemcpyAsync(&flags, c->status, sizeof(int), cudaMemcpyDeviceToHost, M->stream));
  CK(cudaEventRecord(M->ev1, M->stream));
  CK(cudaStreamSynchronize(M->stream));
  cudaEventElapsedTime(&g_last_ms, M->ev0, M->ev1);
  g_last_launches = g_launches + t_serve_launches - served;
  if (flags) {
    llmq_set_error(LLMQ_ERR_CUDA, "%s: the paged cache reported flags 0x%x", fn, flags);
    return 0;
  }
  c->broken = false;
  for (int i = 0; i < n_active; ++i) {
    const int b = active[i];
    for (int k = 0; k < need[b]; ++k) c->pages[b].push_back(c->free_list[c->head_h++]);
    c->len[b] += added[b];
    ids[b] = drawn[i];
  }
  return 1;
}

// No C++ exception leaves a C entry.
template <typename F>
auto guarded(const char *fn, F f, decltype(f()) failed) -> decltype(f()) {
  try {
    return f();
  } catch (...) {
    llmq_set_error(LLMQ_ERR_OOM, "%s: host allocation failed", fn);
    return failed;
  }
}

}  // namespace

extern "C" LLMQ_API int q_llama_decode_batch_sample(const QLlamaModel *m, LlamaKV **kvs, const int *tokens, int B,
                                                    const LlmqSampling *s, int *ids) {
  const char *fn = "q_llama_decode_batch_sample";
  if (B <= 0 || !ids || !s || !s->u) {
    llmq_set_error(LLMQ_ERR_ARG, "%s: bad arguments", fn);
    return LLMQ_ERR_ARG;
  }
  if (g_tp.world > 1) {
    llmq_set_error(LLMQ_ERR_STATE, "%s: not under tensor parallelism", fn);
    return LLMQ_ERR_STATE;
  }
  if (!guarded(fn, [&] { return decode_rows(m, kvs, tokens, B, nullptr, ids, s); }, 0)) return q_llama_last_error();
  for (int b = 0; b < B; ++b) kvs[b]->len = kvs[b]->len + 1;
  return LLMQ_OK;
}

extern "C" LLMQ_API LlmqPagedCache *q_llama_paged_create(const QLlamaModel *m, int n_pages, int page_size, int max_seqs,
                                                         int dtype) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  return guarded("q_llama_paged_create", [&] { return paged_create(m, n_pages, page_size, max_seqs, dtype); },
                 static_cast<LlmqPagedCache *>(nullptr));
}

extern "C" LLMQ_API void q_llama_paged_free(LlmqPagedCache *handle) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  if (!handle) return;
  int cur = -1;
  cudaGetDevice(&cur);
  LlmqPagedCache *c = find_paged(handle, "q_llama_paged_free", true);
  if (c) {
    auto &v = c->model->paged;
    v.erase(std::remove(v.begin(), v.end(), c), v.end());
    cudaStreamSynchronize(c->model->stream);
    release_paged(c);
  }
  if (cur >= 0) cudaSetDevice(cur);
}

extern "C" LLMQ_API int q_llama_paged_len(const LlmqPagedCache *handle, int seq) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const LlmqPagedCache *c = find_paged(handle, "q_llama_paged_len", false);
  if (!c) return -1;
  if (seq < 0 || seq >= c->max_seqs) {
    llmq_set_error(LLMQ_ERR_ARG, "q_llama_paged_len: sequence %d outside [0, %d)", seq, c->max_seqs);
    return -1;
  }
  return c->len[(size_t)seq];
}

extern "C" LLMQ_API int q_llama_paged_free_pages(const LlmqPagedCache *handle) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  const LlmqPagedCache *c = find_paged(handle, "q_llama_paged_free_pages", false);
  return c ? static_cast<int>(c->free_list.size()) - c->head_h : -1;
}

extern "C" LLMQ_API int q_llama_paged_reset(LlmqPagedCache *handle, int seq) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  LlmqPagedCache *c = find_paged(handle, "q_llama_paged_reset", true);
  if (!c) return q_llama_last_error();
  if (seq < 0 || seq >= c->max_seqs) {
    llmq_set_error(LLMQ_ERR_ARG, "q_llama_paged_reset: sequence %d outside [0, %d)", seq, c->max_seqs);
    return LLMQ_ERR_ARG;
  }
  if (c->broken) {
    llmq_set_error(LLMQ_ERR_STATE, "q_llama_paged_reset: an earlier step failed on the GPU");
    return LLMQ_ERR_STATE;
  }
  return guarded("q_llama_paged_reset", [&] { return paged_reset(c, seq); }, 0) ? LLMQ_OK : q_llama_last_error();
}

extern "C" LLMQ_API int q_llama_paged_step(const QLlamaModel *m, LlmqPagedCache *handle, const int *added,
                                           const int *tokens, const LlmqSampling *s, int *ids, Tensor *logits) {
  std::lock_guard<std::recursive_mutex> lk(g_mu);
  LlmqPagedCache *c = find_paged(handle, "q_llama_paged_step", true);
  if (!c) return q_llama_last_error();
  return guarded("q_llama_paged_step", [&] { return paged_step(m, c, added, tokens, s, ids, logits); }, 0)
             ? LLMQ_OK
             : q_llama_last_error();
}
