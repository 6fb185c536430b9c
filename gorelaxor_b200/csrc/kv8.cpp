// grx_kv8_* and grx_logprobs: the arguments' checks and the launches. All
// take device memory and a stream, allocate nothing, and leave the caller's
// current device as it was.
#include "kv8.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include "host.h"
#include "logp.h"

using namespace grx;

namespace {

constexpr int kMaxDevices = 64;
std::atomic<bool> g_ready[kMaxDevices];

// Makes `dev` the current device for a call, its kernels set up, and puts
// the caller's back on every return path.
struct OnDevice {
  int prev = -1, rc = GRX_OK;
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (dev < 0 || dev >= kMaxDevices) {
      rc = fail(GRX_ENODEV, "no CUDA device " + std::to_string(dev));
    } else if (!g_ready[dev].load(std::memory_order_acquire)) {
      rc = device_init(dev);  // leaves dev current
      if (rc == GRX_OK) g_ready[dev].store(true, std::memory_order_release);
    } else if (prev != dev && cudaSetDevice(dev) != cudaSuccess) {
      rc = fail(GRX_ECUDA, "cudaSetDevice(" + std::to_string(dev) + ")");
    } else if (prev == dev) {
      prev = -1;  // nothing to put back
    }
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

int type_size(int type) { return type == GRX_F32 ? 4 : type == GRX_F16 || type == GRX_BF16 ? 2 : 0; }

bool at_multiple(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The cache and the sequences as the kernels take them; `host`: the arrays
// are host memory, and neither the cache's nor the rotation's are looked at.
int args_of(const char* who, const grx_kv8* kv, const grx_kv8_seqs* s, bool host, Kv8Args* out) {
  const std::string w = who;
  if (!kv || !s) return fail(GRX_EINVAL, w + ": null argument");
  if (kv->page_tokens != 16 && kv->page_tokens != 32 && kv->page_tokens != 64)
    return fail(GRX_EINVAL, w + ": pages of " + std::to_string(kv->page_tokens) + " tokens (16, 32 or 64)");
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return fail(GRX_EINVAL, w + ": heads of " + std::to_string(kv->head_dim) + " values (64 or 128)");
  if (kv->kv_heads < 1 || kv->kv_heads > 1024 || kv->pages < 1)
    return fail(GRX_EINVAL, w + ": " + std::to_string(kv->kv_heads) + " heads, " + std::to_string(kv->pages) + " pages");
  if (!host) {
    if (!kv->k || !kv->v || !kv->scale) return fail(GRX_EINVAL, w + ": null cache");
    if (!at_multiple(kv->k, 16) || !at_multiple(kv->v, 16) || !at_multiple(kv->scale, 8))
      return fail(GRX_EINVAL, w + ": the cache's bytes begin at 16-byte boundaries, its scales at one of 8");
  }
  if (s->n < 0 || s->n > 65535) return fail(GRX_EINVAL, w + ": " + std::to_string(s->n) + " sequences (up to 65535)");
  if (s->n > 0 && (!s->table || !s->len)) return fail(GRX_EINVAL, w + ": null table or lengths");
  if (s->table_width < 1 || s->table_width > INT32_MAX / 64)
    return fail(GRX_EINVAL, w + ": a table " + std::to_string(s->table_width) + " pages wide");
  if (s->rows < 0 || s->max_len < 0 || s->max_new < 0 || (!s->row0 && s->rows < s->n))
    return fail(GRX_EINVAL, w + ": " + std::to_string(s->rows) + " rows for " + std::to_string(s->n) + " sequences");
  if (!s->row0 && s->max_new != 1)
    return fail(GRX_EINVAL, w + ": max_new is 1 where each sequence has one row (row0 NULL)");
  Kv8Args a;
  a.k = kv->k;
  a.v = kv->v;
  a.scale = kv->scale;
  a.pages = kv->pages;
  a.plog = kv->page_tokens == 16 ? 4 : kv->page_tokens == 32 ? 5 : 6;
  a.heads = kv->kv_heads;
  a.n = s->n;
  a.width = s->table_width;
  a.rows = s->rows;
  a.max_new = s->max_new;
  a.max_len = s->max_len;
  a.table = s->table;
  a.len = s->len;
  a.row0 = s->row0;
  a.first = s->first;
  if (s->rope_mode != GRX_ROPE_NONE) {
    if (s->rope_mode != GRX_ROPE_PAIRS && s->rope_mode != GRX_ROPE_HALVES)
      return fail(GRX_EINVAL, w + ": rope_mode " + std::to_string(s->rope_mode));
    if (s->rope_positions < 1) return fail(GRX_EINVAL, w + ": a rotation of no positions");
    if (!host && (!s->rope || !at_multiple(s->rope, 16)))
      return fail(GRX_EINVAL, w + ": the rotation's table begins at a 16-byte boundary");
    a.rope = s->rope;
    a.rope_positions = s->rope_positions;
    a.rope_mode = s->rope_mode;
  }
  a.status = s->status;
  *out = a;
  return GRX_OK;
}

int rows_of(const char* who, const char* what, int type, const void* p, int64_t row, int64_t head, Kv8Rows* out) {
  if (!type_size(type)) return fail(GRX_EINVAL, std::string(who) + ": type " + std::to_string(type));
  if (!at_multiple(p, size_t(type_size(type))) || row < 0 || head < 0)
    return fail(GRX_EINVAL, std::string(who) + ": " + what + ": a stride below 0, or values off their own size's boundary");
  out->p = p;
  out->row = row;
  out->head = head;
  return GRX_OK;
}

bool nothing(const Kv8Args& a) { return a.n == 0 || a.rows == 0 || a.max_new == 0; }

int launched(const char* who, cudaError_t e) {
  if (e != cudaSuccess) return fail(GRX_ECUDA, std::string(who) + ": launch: " + cudaGetErrorString(e));
  return GRX_OK;
}

}  // namespace

extern "C" {

int grx_kv8_append(const grx_kv8* kv, const grx_kv8_seqs* s, int type, const void* k, int64_t k_row, int64_t k_head,
                   const void* v, int64_t v_row, int64_t v_head, void* stream) {
  const char* who = "grx_kv8_append";
  Kv8Args a;
  Kv8Rows kr, vr;
  int rc = args_of(who, kv, s, false, &a);
  if (!rc) rc = rows_of(who, "keys", type, k, k_row, k_head, &kr);
  if (!rc) rc = rows_of(who, "values", type, v, v_row, v_head, &vr);
  if (rc) return rc;
  if (nothing(a)) return GRX_OK;
  if (!k || !v) return fail(GRX_EINVAL, "grx_kv8_append: null keys or values");
  if (a.n * kv8_append_pages(a.max_new, kv->page_tokens) * 2 * a.heads > INT32_MAX)
    return fail(GRX_ERANGE, "grx_kv8_append: too many pages for one call; append fewer tokens at a time");
  const OnDevice on(kv->device);
  if (on.rc) return on.rc;
  return launched(who, launch_kv8_append(a, kv->head_dim, type, kr, vr, static_cast<cudaStream_t>(stream)));
}

int grx_kv8_read(const grx_kv8* kv, const grx_kv8_seqs* s, int type, void* k, int64_t k_row, int64_t k_head, void* v,
                 int64_t v_row, int64_t v_head, void* stream) {
  const char* who = "grx_kv8_read";
  Kv8Args a;
  Kv8Rows kr, vr;
  int rc = args_of(who, kv, s, false, &a);
  if (!rc) rc = rows_of(who, "keys", type, k, k_row, k_head, &kr);
  if (!rc) rc = rows_of(who, "values", type, v, v_row, v_head, &vr);
  if (rc) return rc;
  a.rope_mode = GRX_ROPE_NONE;  // stored keys are turned already
  if (nothing(a) || (!k && !v)) return GRX_OK;
  const OnDevice on(kv->device);
  if (on.rc) return on.rc;
  return launched(who, launch_kv8_read(a, kv->head_dim, type, kr, vr, static_cast<cudaStream_t>(stream)));
}

int grx_kv8_attend(const grx_kv8* kv, const grx_kv8_seqs* s, int type, int heads, const void* q, int64_t q_row,
                   int64_t q_head, float scale, int window, void* out, int64_t out_row, int64_t out_head, float* lse,
                   void* stream) {
  const char* who = "grx_kv8_attend";
  Kv8Args a;
  Kv8Attend t;
  int rc = args_of(who, kv, s, false, &a);
  if (!rc) rc = rows_of(who, "queries", type, q, q_row, q_head, &t.q);
  if (!rc) rc = rows_of(who, "outputs", type, out, out_row, out_head, &t.out);
  if (rc) return rc;
  if (heads < 1 || heads % a.heads != 0 || heads / a.heads > 1024)
    return fail(GRX_EINVAL, "grx_kv8_attend: " + std::to_string(heads) + " query heads over " + std::to_string(a.heads) +
                                " key heads");
  if (window < 0 || !std::isfinite(scale)) return fail(GRX_EINVAL, "grx_kv8_attend: window or scale");
  if (!at_multiple(lse, 4)) return fail(GRX_EINVAL, "grx_kv8_attend: lse off a 4-byte boundary");
  if (nothing(a)) return GRX_OK;
  if (!q || !out) return fail(GRX_EINVAL, "grx_kv8_attend: null queries or outputs");
  // blocks of one key head's queries, eight at least, up to sixteen to a stretch of keys
  if ((int64_t(a.max_new) * (heads / a.heads) / 8 + 1) * a.n * a.heads * 16 > INT32_MAX)
    return fail(GRX_ERANGE, "grx_kv8_attend: too many queries for one call; attend in parts");
  t.heads = heads;
  t.scale = scale;
  t.window = window;
  t.lse = lse;
  const OnDevice on(kv->device);
  if (on.rc) return on.rc;
  return launched(who, launch_kv8_attend(a, kv->head_dim, type, t, static_cast<cudaStream_t>(stream)));
}

int grx_kv8_check(const grx_kv8* kv, const grx_kv8_seqs* s, int writes) {
  Kv8Args a;
  const int rc = args_of("grx_kv8_check", kv, s, true, &a);
  if (rc) return rc;
  auto bad = [](int i, const std::string& what) {
    return fail(GRX_ERANGE, "grx_kv8_check: sequence " + std::to_string(i) + ": " + what);
  };
  const auto begins = [&](const Kv8Span& sp) { return (sp.len - sp.T) >> a.plog; };  // the first page it appends to
  const auto pages_of = [&](const Kv8Span& sp) { return (sp.len + (1 << a.plog) - 1) >> a.plog; };
  std::vector<std::pair<int, int>> written;  // pages that are appended to, and by which sequence
  for (int i = 0; i < a.n; i++) {
    const Kv8Span sp = kv8_span(a, i);
    if (!sp.ok)
      return bad(i, a.row0 ? "rows " + std::to_string(a.row0[i]) + " to " + std::to_string(a.row0[i + 1]) + ", " +
                                 std::to_string(sp.len) + " tokens"
                           : std::to_string(sp.len) + " tokens");
    for (int b = 0; b < pages_of(sp); b++) {
      const int p = kv8_page(a, i, b);
      if (p < 0)
        return bad(i, "its page " + std::to_string(b) + " is " + std::to_string(a.table[int64_t(i) * a.width + b]) +
                          " of " + std::to_string(a.pages));
      if (writes && sp.len >= sp.T && sp.T > 0 && b >= begins(sp)) written.emplace_back(p, i);
    }
  }
  std::sort(written.begin(), written.end());
  for (size_t j = 1; j < written.size(); j++)
    if (written[j].first == written[j - 1].first)
      return bad(written[j].second, "appends to page " + std::to_string(written[j].first) + ", as sequence " +
                                        std::to_string(written[j - 1].second) + " does");
  if (!written.empty())
    for (int i = 0; i < a.n; i++) {
      const Kv8Span sp = kv8_span(a, i);
      const int whole = sp.T > 0 && sp.len >= sp.T ? begins(sp) : pages_of(sp);
      for (int b = 0; b < whole; b++) {
        const int p = kv8_page(a, i, b);
        const auto w = std::lower_bound(written.begin(), written.end(), std::make_pair(p, 0));
        if (w != written.end() && w->first == p)
          return bad(i, "holds page " + std::to_string(p) + ", which sequence " + std::to_string(w->second) +
                            " appends to");
      }
    }
  return GRX_OK;
}

int grx_logprobs(int device, int type, const void* logits, int rows, int vocab, int64_t row_stride,
                 const int* targets, int top, float* logprob, float* entropy, int* top_ids, float* top_logprobs,
                 void* stream) {
  const char* who = "grx_logprobs";
  if (!type_size(type)) return fail(GRX_EINVAL, "grx_logprobs: type " + std::to_string(type));
  if (rows < 0 || vocab < 1 || vocab == INT32_MAX || row_stride < 0)
    return fail(GRX_EINVAL, "grx_logprobs: " + std::to_string(rows) + " rows of " + std::to_string(vocab));
  if (top < 0 || top > kLogpMaxTop || top > vocab)
    return fail(GRX_EINVAL, "grx_logprobs: " + std::to_string(top) + " alternatives (0 to " +
                                std::to_string(kLogpMaxTop) + ", and of a vocabulary of " + std::to_string(vocab) + ")");
  if (logprob && !targets) return fail(GRX_EINVAL, "grx_logprobs: logprob without targets");
  if (!at_multiple(logits, size_t(type_size(type))) || !at_multiple(targets, 4) || !at_multiple(logprob, 4) ||
      !at_multiple(entropy, 4) || !at_multiple(top_ids, 4) || !at_multiple(top_logprobs, 4))
    return fail(GRX_EINVAL, "grx_logprobs: values off their own size's boundary");
  LogpArgs a;
  a.x = logits;
  a.stride = row_stride;
  a.rows = rows;
  a.vocab = vocab;
  a.top = top_ids || top_logprobs ? top : 0;
  a.targets = targets;
  a.logprob = logprob;
  a.entropy = entropy;
  a.ids = top_ids;
  a.lps = top_logprobs;
  if (rows == 0 || (!logprob && !entropy && a.top == 0)) return GRX_OK;
  if (!logits) return fail(GRX_EINVAL, "grx_logprobs: null logits");
  const OnDevice on(device);
  if (on.rc) return on.rc;
  return launched(who, launch_logp(a, type, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
