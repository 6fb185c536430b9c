// Log probabilities of given tokens, with the entropy of each row and its
// most likely tokens, in one pass over the logits.
//
// With m the row's largest logit (at one index) and the sums over the other
// indices
//   z = Σ e^(x_j − m),   t = Σ (m − x_j)·e^(x_j − m),
// the log probability of token j is (x_j − m) − log1p(z) and the entropy is
// log1p(z) + t/(1 + z). Every term is positive and the 1 is kept apart, so a
// row whose model is sure loses nothing to cancellation.
//
// In the pass each thread keeps the largest value m' of its own and sums over
// all of them, largest included, moved to a new m' once for every few vectors
// (no branch: a branch "only where the largest grows" is taken by some lane
// of nearly every warp). Its sums hold a 1 that hides small terms only where
// m' is about m. The threads with the largest m' are looked at a second time
// anyway, for the most likely tokens, and their sums are then made anew
// without the values equal to m.
//
// The most likely tokens: the `top`-th largest of the threads' m' is a bound
// that the answer does not go below, so only the threads at or above it
// (about `top` of hundreds) have their values looked at again, and the few
// values above the bound are ranked. Values compare as (value, lower index
// first), each as one 64-bit number; NaN counts below −inf.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "logp.h"

namespace grx {

namespace {

constexpr uint32_t FULL = 0xffffffffu;
constexpr float kLog2e = 1.44269504f;
constexpr float kFar = -200.f;  // e^kFar is 0 in 32 bits; stands for −inf where a product with 0 follows
typedef unsigned long long u64;

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float qnan() { return __int_as_float(0x7fc00000); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(__half h) { return __half2float(h); }
__device__ __forceinline__ float wide(__nv_bfloat16 h) { return __bfloat162float(h); }

// A value as a whole number of the same order; −0 as 0, NaN below all.
__device__ __forceinline__ uint32_t order(float x) {
  if (isnan(x)) return 0;
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.f));
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unorder(uint32_t u) {
  if (u == 0) return qnan();
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// (value, lower index first) as one number; 0 is no token.
__device__ __forceinline__ u64 key_of(float x, int i) { return u64(order(x)) << 32 | uint32_t(0x7fffffff - i); }

// A share of a row: its largest value (−inf: none), and the sums over the
// others.
struct Share {
  float m, z, t;
};

// Two shares with m1 >= m2 and e = e^(m2 − m1):
//   z = z1 + e·(1 + z2),   t = t1 + e·(t2 + (m1 − m2)·(1 + z2)).
__device__ __forceinline__ Share join(Share a, Share b) {
  if (b.m > a.m) {
    const Share c = a;
    a = b;
    b = c;
  }
  if (b.m == ninf()) {
    // nothing that counts, unless a NaN is in its sums
    a.z = __fadd_rn(a.z, b.z);
    return a;
  }
  const float d = fmaxf(__fsub_rn(b.m, a.m), kFar), e = ex2(__fmul_rn(d, kLog2e)), n = __fadd_rn(1.f, b.z);
  a.z = __fmaf_rn(e, n, a.z);
  a.t = __fmaf_rn(e, __fmaf_rn(-d, n, b.t), a.t);
  return a;
}

// All 32 lanes' shares; every lane gets the same bits.
__device__ __forceinline__ Share warp_join(Share s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Share b;
    b.m = __shfl_xor_sync(FULL, s.m, o);
    b.z = __shfl_xor_sync(FULL, s.z, o);
    b.t = __shfl_xor_sync(FULL, s.t, o);
    s = threadIdx.x & o ? join(b, s) : join(s, b);
  }
  return s;
}

__device__ __forceinline__ u64 warp_max(u64 k) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(FULL, k, o));
  return k;
}
__device__ __forceinline__ float warp_max(float m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
  return m;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(FULL, v, o));
  return v;
}

// One value into sums over e^(x − m), x <= m (or NaN: the sums become NaN).
__device__ __forceinline__ void add(float& z, float& t, float x, float m) {
  const float d = max_nan(__fsub_rn(x, m), kFar), e = ex2(__fmul_rn(d, kLog2e));
  z = __fadd_rn(z, e);
  t = __fmaf_rn(-d, e, t);
}

// A thread's values: the largest, and z and t over all of them.
struct Run {
  float m = ninf(), z = 0.f, t = 0.f;
};

// Values two by two, the sums in two halves: packed 32-bit operations, each
// half rounded as one alone.
template <int N>
__device__ __forceinline__ void take(Run& r, const float (&x)[N]) {
  float c = r.m;
#pragma unroll
  for (int j = 0; j < N; j++) c = fmaxf(c, x[j]);
  // the sums so far, from r.m to c; without a finite value so far they are 0
  // (or NaN), and without one now they stay that
  const float up = r.m == c ? 0.f : fmaxf(__fsub_rn(r.m, c), kFar), k = ex2(__fmul_rn(up, kLog2e));
  r.t = __fmul_rn(k, __fmaf_rn(-up, r.z, r.t));
  r.z = __fmul_rn(k, r.z);
  r.m = c;
  const float mm = c == ninf() ? 0.f : c;
  if constexpr (N % 2 == 0) {
    f2 z = 0, t = 0;
    const f2 nm = f2dup(-mm), l = f2dup(kLog2e), one = f2dup(-1.f);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const f2 d = f2add(f2make(x[j], x[j + 1]), nm);
      const f2 dc = f2make(max_nan(f2lo(d), kFar), max_nan(f2hi(d), kFar));
      const f2 y = f2mul(dc, l);
      const f2 e = f2make(ex2(f2lo(y)), ex2(f2hi(y)));
      z = f2add(z, e);
      t = f2fma(dc, e, t);
    }
    t = f2mul(t, one);
    r.z = __fadd_rn(r.z, __fadd_rn(f2lo(z), f2hi(z)));
    r.t = __fadd_rn(r.t, __fadd_rn(f2lo(t), f2hi(t)));
  } else {
#pragma unroll
    for (int j = 0; j < N; j++) add(r.z, r.t, x[j], mm);
  }
}

template <class T>
__device__ __forceinline__ void unpack16(uint4 q, float* x) {
  constexpr int V = 16 / sizeof(T);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < V; j++) {
    if constexpr (sizeof(T) == 4)
      x[j] = __uint_as_float(w[j]);
    else if constexpr (std::is_same<T, __half>::value)
      x[j] = __half2float(__ushort_as_half(uint16_t(w[j / 2] >> (16 * (j % 2)))));
    else
      x[j] = bits_f(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
}
template <class T>
__device__ __forceinline__ void load16(const T* p, float* x) {
  unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p)), x);
}

// What the row's outputs are made of, by one thread.
template <class T>
__device__ __forceinline__ void row_out(const LogpArgs& a, int row, const T* x, Share s) {
  // no largest number, no distribution
  const bool fine = isfinite(s.m);
  const float lz = log1pf(s.z);
  if (a.logprob) {
    const int t = a.targets[row];
    a.logprob[row] = fine && t >= 0 && t < a.vocab ? __fsub_rn(__fsub_rn(wide(x[t]), s.m), lz) : qnan();
  }
  if (a.entropy) a.entropy[row] = fine ? __fadd_rn(lz, __fdiv_rn(s.t, __fadd_rn(1.f, s.z))) : qnan();
}

__device__ __forceinline__ void top_out(const LogpArgs& a, int row, int r, u64 key, Share s) {
  if (a.ids) a.ids[int64_t(row) * a.top + r] = 0x7fffffff - int(uint32_t(key));
  if (a.lps)
    a.lps[int64_t(row) * a.top + r] =
        isfinite(s.m) ? __fsub_rn(__fsub_rn(unorder(uint32_t(key >> 32)), s.m), log1pf(s.z)) : qnan();
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <class V>
__device__ __forceinline__ V peer(const V* p, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank));
  V v;
  if constexpr (sizeof(V) == 8)
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at));
  else
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

// ---- a row to a cluster of S blocks of NT threads ----
//
// Bound by the bytes of the logits. Loads are 16 bytes wide from the first
// aligned value on, two to a thread in flight ahead of the two that are
// summed; few rows are split over a
// cluster, whose first block joins the shares through distributed shared
// memory. Three blocks of 512 threads an SM: 107 us for 2048 rows of 100003
// bfloat16 logits (two blocks with four vectors a turn 121, five of 256
// threads 123).
constexpr int kCand = 1024, kBlock = 512, kSmallBlock = 128;

template <class T, int NT>
__global__ void __launch_bounds__(NT, 1536 / NT) k_logp(LogpArgs a, int S) {
  constexpr int V = 16 / sizeof(T), U = 2, NW = NT / 32;
  __shared__ float wm[NW], wn[NW], wz[NW], wt[NW];
  __shared__ u64 wk[NW];
  __shared__ u64 cand[kCand];
  __shared__ u64 best[kLogpMaxTop];
  __shared__ int ncand, nties;
  __shared__ Share mine, whole;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int rank = S > 1 ? int(cluster_rank()) : 0, row = blockIdx.x / S, k = a.top;
  const T* x = static_cast<const T*>(a.x) + int64_t(row) * a.stride;
  const int head = min(a.vocab, int((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / int(sizeof(T)));
  const int nv = (a.vocab - head) / V, tail = a.vocab - head - nv * V;
  const T* xv = x + head;
  const int vb = int(int64_t(nv) * rank / S), ve = int(int64_t(nv) * (rank + 1) / S);
  // the values before and behind the vectors, one to a thread
  const bool in_head = rank == 0 && tid < head, in_tail = rank == S - 1 && tid < tail;
  const int at_tail = a.vocab - tail + tid;
  if (tid == 0) ncand = nties = 0;

  Run r;
  int v = vb + tid;
  if (v + (U - 1) * NT < ve) {
    // the next vectors come while these are summed
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = __ldg(reinterpret_cast<const uint4*>(xv) + v + u * NT);
    for (;;) {
      float f[U * V];
#pragma unroll
      for (int u = 0; u < U; u++) unpack16<T>(raw[u], f + u * V);
      v += U * NT;
      const bool more = v + (U - 1) * NT < ve;
      if (more) {
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = __ldg(reinterpret_cast<const uint4*>(xv) + v + u * NT);
      }
      take(r, f);
      if (!more) break;
    }
  }
  for (; v < ve; v += NT) {
    float f[V];
    load16(xv + int64_t(v) * V, f);
    take(r, f);
  }
  if (in_head) {
    const float f[1] = {wide(x[tid])};
    take(r, f);
  }
  if (in_tail) {
    const float f[1] = {wide(x[at_tail])};
    take(r, f);
  }
  const bool some = vb + tid < ve || in_head || in_tail;
  {
    const float m = warp_max(r.m), n = -warp_max(-r.m);
    if (lane == 0) wm[warp] = m, wn[warp] = n;
  }
  __syncthreads();
  float m = wm[0], least = wn[0];
#pragma unroll
  for (int w = 1; w < NW; w++) m = fmaxf(m, wm[w]), least = fminf(least, wn[w]);
  // the bound: the largest value, or the largest found, bit by bit, that
  // `top` threads reach
  const uint32_t u = order(r.m);
  uint32_t bound = order(m);
  if (k > 1) {
    // what the largest and the least have in common is the bound's too
    const uint32_t ul = order(least), apart = bound ^ ul;
    const int high = apart ? 32 - __clz(apart) : 0;
    bound = high < 32 ? ul >> high << high : 0;
    if (__syncthreads_count(some) < k) bound = 0;  // fewer values than asked for: all
    for (int bit = high - 1; bit >= 0; bit--) {
      const uint32_t c = bound | 1u << bit;
      const int n = __syncthreads_count(some && u >= c);
      if (n >= k) {
        bound = c;
        if (n <= k + 8) break;
      }
    }
  }
  const bool again = some && u >= bound;
  if (tid < k) best[tid] = 0;
  // The chosen threads' values once more, their warp to a thread's: where m
  // is among them, their sums without the values equal to it (so no number
  // depends on `top`); and the values that reach the bound.
  const bool owner = some && r.m == m;
  float z = 0.f, t = 0.f;
  int ties = 0;
  // (bound 0: every value, those that are no number too)
  const float reach = unorder(bound);
  auto look = [&](float f, int i, bool sums) {
    if (sums) {
      if (f == m)
        ties++;
      else if (f != ninf())
        add(z, t, f, m);
    }
    if (f >= reach || bound == 0) {
      const int p = atomicAdd(&ncand, 1);
      if (p < kCand) cand[p] = key_of(f, i);
    }
  };
  if (!owner) {
    const float d = r.m == ninf() ? 0.f : fmaxf(__fsub_rn(r.m, m), kFar), e = ex2(__fmul_rn(d, kLog2e));
    t = __fmul_rn(e, __fmaf_rn(-d, r.z, r.t));
    z = __fmul_rn(e, r.z);
  }
  if (again && in_head) look(wide(x[tid]), tid, owner);
  if (again && in_tail) look(wide(x[at_tail]), at_tail, owner);
  const uint32_t owners = __ballot_sync(FULL, owner);
  for (uint32_t chosen = __ballot_sync(FULL, again); chosen; chosen &= chosen - 1) {
    const int j = __ffs(chosen) - 1;
    const bool sums = owners >> j & 1;
    for (int w = vb + warp * 32 + j + lane * NT; w < ve; w += 32 * NT) {
      float f[V];
      load16(xv + int64_t(w) * V, f);
#pragma unroll
      for (int e = 0; e < V; e++) look(f[e], head + w * V + e, sums);
    }
  }
  z = warp_sum(z);
  t = warp_sum(t);
  if (ties) atomicAdd(&nties, ties);
  if (lane == 0) {
    wz[warp] = z;
    wt[warp] = t;
  }
  __syncthreads();
  if (warp == 0) {
    z = warp_sum(lane < NW ? wz[lane] : 0.f);
    t = warp_sum(lane < NW ? wt[lane] : 0.f);
    // equals of m but one count 1 each, with no gap; −inf counts nothing
    if (lane == 0) mine = Share{m, m == ninf() ? z : __fadd_rn(z, float(max(nties, 1) - 1)), t};
  }
  if (k) {
    const int n = ncand, all = (ve - vb) * V + (rank == 0 ? head : 0) + (rank == S - 1 ? tail : 0);
    if (n >= min(k, all) && n <= kCand) {
      for (int c = tid; c < n; c += NT) {
        const u64 mk = cand[c];
        int above = 0;
        for (int d = 0; d < n; d++) above += cand[d] > mk;
        if (above < k) best[above] = mk;
      }
    } else {
      // More equals than the list takes (or values that are no number among
      // the threads' counted): the largest below the last, k times.
      u64 last = ~u64(0);
      for (int c = 0; c < k; c++) {
        u64 q = 0;
        auto see = [&](float f, int i) {
          const u64 y = key_of(f, i);
          if (y < last && y > q) q = y;
        };
        if (in_head) see(wide(x[tid]), tid);
        if (in_tail) see(wide(x[at_tail]), at_tail);
        for (int w = vb + tid; w < ve; w += NT) {
          float f[V];
          load16(xv + int64_t(w) * V, f);
#pragma unroll
          for (int e = 0; e < V; e++) see(f[e], head + w * V + e);
        }
        q = warp_max(q);
        if (lane == 0) wk[warp] = q;
        __syncthreads();
        last = 0;
        for (int w = 0; w < NW; w++) last = max(last, wk[w]);
        __syncthreads();
        if (tid == 0) best[c] = last;
      }
    }
  }
  if (S == 1) {
    __syncthreads();
    if (tid == 0) row_out(a, row, x, mine);
    if (tid < k) top_out(a, row, tid, best[tid], mine);
    return;
  }
  cluster_sync();
  if (rank == 0) {
    if (warp == 0) {
      Share s = {ninf(), 0.f, 0.f};
      if (lane < S) s = Share{peer(&mine.m, lane), peer(&mine.z, lane), peer(&mine.t, lane)};
      s = warp_join(s);
      if (lane == 0) whole = s;
    }
    for (int j = tid; j < S * k; j += NT) cand[j] = peer(&best[j % k], j / k);
  }
  cluster_sync();  // no block leaves while its shared memory is read
  if (rank != 0) return;
  if (tid == 0) row_out(a, row, x, whole);
  for (int j = tid; j < S * k; j += NT) {
    const u64 mk = cand[j];
    int above = 0;
    for (int d = 0; d < S * k; d++) above += cand[d] > mk;
    if (mk && above < k) top_out(a, row, above, mk, whole);
  }
}

// ---- short rows: a warp each, the row in its registers ----
//
// The bound is what `top` lanes' largest values reach. From 28 alternatives on
// the search for it stops at the first bit that all 32 lanes reach, which
// half of a usual row passes: the list is then too short and the row is scanned
// `top` times. 24000 rows of 1030 float32 values: 25 us for one alternative, 77
// for 24, 495 for 28.
constexpr int kWarpCand = 128, kRowsPerBlock = 8;

template <class T, int NE>
__global__ void __launch_bounds__(32 * kRowsPerBlock, NE > 48 ? 2 : 4) k_logp_warp(LogpArgs a) {
  __shared__ u64 cands[kRowsPerBlock][kWarpCand];
  __shared__ int counts[kRowsPerBlock];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, k = a.top;
  const int64_t row64 = int64_t(blockIdx.x) * kRowsPerBlock + warp;
  if (row64 >= a.rows) return;
  const int row = int(row64);
  const T* x = static_cast<const T*>(a.x) + row64 * a.stride;
  // values behind the row are −inf: they count nothing anywhere but among
  // the candidates, which look at the index
  const int whole = a.vocab / 32, rest = a.vocab % 32;
  float f[NE];
#pragma unroll
  for (int j = 0; j < NE; j++) f[j] = j < whole || (j == whole && lane < rest) ? wide(x[lane + 32 * j]) : ninf();
  float mine = f[0];
#pragma unroll
  for (int j = 1; j < NE; j++) mine = fmaxf(mine, f[j]);
  if (isnan(mine)) mine = ninf();
  const float m = warp_max(mine);
  Share s = {m, 0.f, 0.f};
  int ties = 0, at = 0x7fffffff;
  {
    f2 z = 0, t = 0;
    const f2 nm = f2dup(-m), l2e = f2dup(kLog2e);
#pragma unroll
    for (int j = NE - 2; j >= 0; j -= 2) {
      if (j > whole) continue;
      const f2 d = f2add(f2make(f[j], f[j + 1]), nm);
      const f2 dc = f2make(max_nan(f2lo(d), kFar), max_nan(f2hi(d), kFar)), y = f2mul(dc, l2e);
      float e0 = ex2(f2lo(y)), e1 = ex2(f2hi(y));
      if (f[j + 1] == m) e1 = 0.f, ties++, at = lane + 32 * (j + 1);
      if (f[j] == m) e0 = 0.f, ties++, at = lane + 32 * j;
      const f2 e = f2make(e0, e1);
      z = f2add(z, e);
      t = f2fma(dc, e, t);
    }
    s.z = __fadd_rn(f2lo(z), f2hi(z));
    s.t = -__fadd_rn(f2lo(t), f2hi(t));
  }
  s.z = warp_sum(s.z);
  s.t = warp_sum(s.t);
  ties = __reduce_add_sync(FULL, ties);
  s.z = __fadd_rn(s.z, float(max(ties, 1) - 1));
  if (lane == 0) row_out(a, row, x, s);
  if (k == 0) return;
  if (k == 1 && isfinite(m)) {
    at = __reduce_min_sync(FULL, at);
    if (lane == 0) top_out(a, row, 0, key_of(m, at), s);
    return;
  }
  const uint32_t u = order(mine);
  uint32_t bound = 0;
  for (int bit = 31; bit >= 0; bit--) {
    const uint32_t c = bound | 1u << bit;
    const int n = __popc(__ballot_sync(FULL, lane < a.vocab && u >= c));
    if (n >= k) {
      bound = c;
      if (n <= k + 4) break;
    }
  }
  if (lane == 0) counts[warp] = 0;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < NE; j++) {
    const int i = lane + 32 * j;
    if (i < a.vocab && order(f[j]) >= bound) {
      const int p = atomicAdd(&counts[warp], 1);
      if (p < kWarpCand) cands[warp][p] = key_of(f[j], i);
    }
  }
  __syncwarp();
  const int n = counts[warp];
  if (n >= k && n <= kWarpCand) {
    for (int c = lane; c < n; c += 32) {
      const u64 mk = cands[warp][c];
      int above = 0;
      for (int d = 0; d < n; d++) above += cands[warp][d] > mk;
      if (above < k) top_out(a, row, above, mk, s);
    }
  } else {
    u64 last = ~u64(0);
    for (int r = 0; r < k; r++) {
      u64 q = 0;
#pragma unroll
      for (int j = 0; j < NE; j++) {
        const int i = lane + 32 * j;
        const u64 y = i < a.vocab ? key_of(f[j], i) : 0;
        if (y < last && y > q) q = y;
      }
      last = warp_max(q);
      if (lane == 0) top_out(a, row, r, last, s);
    }
  }
}

constexpr int kSMs = 148;

template <class T, int NT>
cudaError_t rows_t(const LogpArgs& a, cudaStream_t st) {
  // few rows: up to eight blocks to a row, each with a few vectors a thread
  int S = 1;
  while (S < 8 && int64_t(a.rows) * S < 2 * kSMs && a.vocab >= 2 * S * NT * int(16 / sizeof(T))) S *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows) * S);
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(S);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_logp<T, NT>, a, S);
}

template <class T, int NE>
void warp_rows(const LogpArgs& a, cudaStream_t st) {
  k_logp_warp<T, NE><<<unsigned((int64_t(a.rows) + kRowsPerBlock - 1) / kRowsPerBlock), 32 * kRowsPerBlock, 0, st>>>(a);
}

// Rows of up to 2048 values: a warp each, with the least multiple of 8 values
// a lane that holds one.
template <class T, int NE = 8>
cudaError_t logp_t(const LogpArgs& a, cudaStream_t st) {
  if constexpr (NE <= 64) {
    if (a.vocab > 32 * NE) return logp_t<T, NE + 8>(a, st);
    warp_rows<T, NE>(a, st);
    return cudaGetLastError();
  } else {
    // A block's exchanges take about 6 us whatever the row's length: many
    // short rows go to more, smaller blocks. 4000 rows of float32 values, us
    // with 512 threads and with 128: of 4000 values 64 and 27, of 16000 89
    // and 68, of 32000 123 and 125. 400 rows of 4000: 12 and 11, of 32000 15
    // and 19; up to 32 rows 512 threads are the faster at any length.
    return a.vocab <= 24 * 1024 && a.rows >= 2 * kSMs ? rows_t<T, kSmallBlock>(a, st) : rows_t<T, kBlock>(a, st);
  }
}

}  // namespace

cudaError_t launch_logp(const LogpArgs& a, int type, cudaStream_t st) {
  const cudaError_t e = type == 0   ? logp_t<float>(a, st)
                        : type == 1 ? logp_t<__half>(a, st)
                                    : logp_t<__nv_bfloat16>(a, st);
  if (e != cudaSuccess) cudaGetLastError();  // returned: a later launch must not find it as its own
  return e;
}

}  // namespace grx
