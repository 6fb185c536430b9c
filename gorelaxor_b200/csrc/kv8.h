// The 8-bit paged cache: its index arithmetic, shared by the kernels
// (k_kv8.cu) and the host's checks (kv8.cpp), and the kernels' launchers.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#ifdef __CUDACC__
#define KV8_FN __host__ __device__ __forceinline__
#else
#define KV8_FN inline
#endif

namespace grx {

// grx_kv8 and grx_kv8_seqs as the kernels take them.
struct Kv8Args {
  int8_t* k = nullptr;  // [pages][heads][page][head_dim]
  int8_t* v = nullptr;
  float* scale = nullptr;  // [pages][heads][2]: keys, values
  int pages = 0, plog = 4, heads = 0;  // plog: log2 of a page's tokens
  int n = 0, width = 0, rows = 0, max_new = 1, max_len = 0;
  const int *table = nullptr, *len = nullptr, *row0 = nullptr, *first = nullptr;
  int len_add = 0;  // tokens of sequence i: len[i] + len_add
  const float* rope = nullptr;
  int rope_positions = 0, rope_mode = 0;
  int* status = nullptr;
};

// The rows of one sequence in this call: rows row .. row + T − 1 stand at
// the positions len − T .. len − 1 (a lone position of −1, in a call of one
// row for each sequence, is a slot that holds nothing).
struct Kv8Span {
  int row, T, len;
  bool ok;
};

// Every bound that a row number or a position is used with later follows
// from `ok`: 0 <= row, row + T <= rows, T <= max_new, the positions below
// width pages and, with a rotation, below the table's positions.
KV8_FN Kv8Span kv8_span(const Kv8Args& a, int i) {
  Kv8Span s;
  s.len = a.len[i] + a.len_add;
  if (a.row0) {
    s.row = a.row0[i];
    const int end = a.row0[i + 1];
    s.ok = s.row >= 0 && end >= s.row && end <= a.rows && end - s.row <= a.max_new && s.len >= end - s.row;
    s.T = s.ok ? end - s.row : 0;
  } else {
    s.row = i;
    s.T = 1;
    s.ok = i < a.rows && s.len >= 0;
  }
  s.ok = s.ok && s.len <= (int64_t(a.width) << a.plog) && (a.rope_mode == 0 || s.len <= a.rope_positions);
  return s;
}

// The page of a sequence's block b (0 <= b < width), or −1 where the
// table's entry is no page.
KV8_FN int kv8_page(const Kv8Args& a, int i, int b) {
  const int p = a.table[int64_t(i) * a.width + b];
  return p >= 0 && p < a.pages ? p : -1;
}

// Pages that max_new tokens of a sequence can touch.
KV8_FN int64_t kv8_append_pages(int max_new, int page) { return (int64_t(max_new) + page - 2) / page + 1; }
// The group of `threads` threads that thread `thread` of block `block` (of
// 256 threads) belongs to. Groups are fewer than 2^31 (the entry point
// refuses more); their threads need not be, so those are never counted.
KV8_FN uint32_t kv8_append_group(uint32_t block, uint32_t thread, int threads) {
  return block * uint32_t(256 / threads) + thread / uint32_t(threads);
}
// Blocks of 256 threads for `groups` groups of `threads` threads.
KV8_FN uint32_t kv8_append_grid(int64_t groups, int threads) {
  return uint32_t((groups + 256 / threads - 1) / (256 / threads));
}

// Rows of keys, values or queries in memory: element e of head h of row r
// is at r·row + h·head + e.
struct Kv8Rows {
  const void* p = nullptr;
  int64_t row = 0, head = 0;
};

struct Kv8Attend {
  Kv8Rows q, out;    // out.p is written
  int heads = 0;     // query heads, a multiple of the cache's
  float scale = 0;
  int window = 0;
  float* lse = nullptr;  // [rows][heads]
  // Q8_0 blocks of the output besides (float32 outputs may be absent then):
  // values [rows][heads·head_dim], scales twice as k_q8's products read them
  int8_t* q8 = nullptr;
  float2* q8s = nullptr;
};

// type: 0 float32, 1 float16, 30 bfloat16 (grx.h's GRX_F32 …).
cudaError_t launch_kv8_append(const Kv8Args& a, int head_dim, int type, const Kv8Rows& k, const Kv8Rows& v,
                              cudaStream_t st);
cudaError_t launch_kv8_read(const Kv8Args& a, int head_dim, int type, const Kv8Rows& k, const Kv8Rows& v,
                            cudaStream_t st);
cudaError_t launch_kv8_attend(const Kv8Args& a, int head_dim, int type, const Kv8Attend& t, cudaStream_t st);
// Copies the pages from[j] to to[j] of `layers` caches that lie one behind
// the other (a is the first).
cudaError_t launch_kv8_copy_pages(const Kv8Args& a, int head_dim, int layers, const int* from, const int* to, int count,
                                  cudaStream_t st);
// launch_kv8_attend's form for many queries of a sequence to a key head
// (k_kv8_prompt.cu).
cudaError_t launch_kv8_prompt(const Kv8Args& a, int head_dim, int type, const Kv8Attend& t, cudaStream_t st);
void kv8_prompt_init();
void kv8_kernels_init();

}  // namespace grx
