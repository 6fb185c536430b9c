// The 8-bit paged key/value cache: appending tokens to it (with the position
// rotation of the keys), reading them back, and attention over it.
//
// A page holds the keys and values of `page` tokens for every head,
// [pages][heads][page][head_dim] bytes each, and two scales per page and
// head; a byte q stands for q·scale. All three kernels take rows through
// kv8_span and pages through kv8_page (kv8.h), which bound every access; a
// sequence or page that does not fit is left out and reported.
#include <cuda_runtime.h>
#include <cuda_bf16.h>

#include <algorithm>

#include "kv8.cuh"

namespace grx {

namespace {

__device__ __forceinline__ void narrow(float x, float* p) { *p = x; }
__device__ __forceinline__ void narrow(float x, __half* p) { *p = __float2half_rn(x); }
__device__ __forceinline__ void narrow(float x, __nv_bfloat16* p) { *p = __float2bfloat16_rn(x); }

// ------------------------------------------------------------- append ----
//
// A unit is one (sequence, page it writes, head, keys or values): G threads
// that hold the page's new values, find the largest magnitude a, and set
// s' = max(s, a/127); where that grew, what the page held becomes
// rne(q·s/s'); the new values become rne(x/s'). No two units share a byte or
// a scale, so there are no atomics and no order.
//
// The definition's rotations and quotients are exact to 64 bits: a value
// next to a rounding border goes to one or the other side by less than 32
// bits hold, a whole step of the page's scale. They are computed in 32 bits,
// which is off by less than 3e-5 of a step (127 steps times 3.4·2^-24), and
// where a value comes within 4e-5 of a border (one in 12000) it is formed
// again in 64 bits and compared with the border, (k ± 1/2)·s', itself: that
// product is exact. The scale's largest magnitude likewise: the values within
// 2^-19 of the largest are formed again in 64 bits (not rotated ones: they
// are exact). Pages of very small or very large numbers (kTiny, kHuge) take
// 64 bits throughout.
//
// A thread holds at most kItems items of eight values: two groups of four
// that the rotation pairs with each other. Bound by latency for single
// tokens: 256 sequences' in 7 us. 12000 tokens of 24 prompts, 8 heads of 128,
// bfloat16: 46 us, 1.7 TB/s of rows and pages, bound by each page's chain
// (rows, exchange, rescaling, rounding) at three blocks an SM: with four, and
// fewer registers, the whole case takes 84 us instead of 67, with a tenth
// fewer instructions (packed roundings) the same.
constexpr int kItems = 4;
constexpr float kNear = 0.49996f;
constexpr float kTiny = 1e-30f, kHuge = 1e37f;

// Element j (0..7) of an item in 64 bits: elements e0 .. e0 + 3 and e1 ..
// e1 + 3 of a row, rotated by the angles at cs.
template <class T>
__device__ __forceinline__ double value64(const T* src, int e0, int e1, int mode, const float* cs, int j) {
  const auto at = [&](int n) { return double(wide(src[n < 4 ? e0 + n : e1 + n - 4])); };
  if (mode == ROPE_NONE) return at(j);
  const int n = mode == ROPE_PAIRS ? j >> 1 : j & 3, second = mode == ROPE_PAIRS ? j & 1 : j >> 2;
  const double xa = at(mode == ROPE_PAIRS ? 2 * n : n), xb = at(mode == ROPE_PAIRS ? 2 * n + 1 : n + 4);
  const double cc = cs[2 * n], ss = cs[2 * n + 1];
  // the products are exact, so one rounding
  return second ? __fma_rn(xa, ss, xb * cc) : __fma_rn(xa, cc, -(xb * ss));
}
// rne(x/s) for a quotient within a step of k: x against the borders of k.
__device__ __forceinline__ int settle(double x, double s, int k) {
  const double up = (k + 0.5) * s, dn = (k - 0.5) * s;
  if (x > up || (x == up && (k & 1))) return k + 1;
  if (x < dn || (x == dn && (k & 1))) return k - 1;
  return k;
}
__device__ __noinline__ double divided(double x, double y) { return x / y; }
// |x|/127 in 32 bits (NaN for what is not finite): the quotient's rounding,
// which a product with 1/127 gives but where it lies on a border as far as 64
// bits tell.
__device__ __forceinline__ float over127(double x) {
  const double m = fabs(x), q = m * (1.0 / 127.0), e = q * 0x1p-51;
  const float lo = float(q - e), hi = float(q + e);
  if (!isfinite(m)) return __int_as_float(0x7fc00000);
  return lo == hi ? lo : float(divided(m, 127.0));
}
// rne(x/s) where neither is known to be in the range of 32-bit reciprocals.
__device__ __noinline__ int rounded64(double x, float s) { return max(-127, min(127, __double2int_rn(x / double(s)))); }

// Four floats n + 1.5·2^23 as bytes n.
__device__ __forceinline__ uint32_t low_bytes(const float* t) {
  return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040),
                     __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
}
// x·r rounded, as n + 1.5·2^23, and whether a border is near.
__device__ __forceinline__ float rounded(float x, float r, bool* near) {
  const float t = __fmaf_rn(x, r, MAGIC);
  *near = fabsf(__fmaf_rn(x, r, -__fsub_rn(t, MAGIC))) > kNear;
  return t;
}

// Four signed bytes times s/s1 (about r), rounded.
__device__ __forceinline__ uint32_t scaled_bytes(uint32_t q, float r, float s, float s1, bool slow) {
  const uint32_t u = q ^ 0x80808080u;
  float t[4];
  uint32_t redo = slow ? 15 : 0;
#pragma unroll
  for (int k = 0; k < 4; k++) {
    bool near;
    t[k] = rounded(__fsub_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 | k)), 8388736.f), r, &near);
    if (near) redo |= 1 << k;
  }
  uint32_t w = low_bytes(t);
  for (; redo; redo &= redo - 1) {
    const int at = 8 * (__ffs(redo) - 1);
    const double x = double(int8_t(q >> at)) * double(s);
    const int v = slow ? rounded64(x, s1) : settle(x, double(s1), int8_t(w >> at));
    w = (w & ~(255u << at)) | uint32_t(v & 255) << at;
  }
  return w;
}

// Eight values of a row as they are in memory.
template <class T>
struct Raw {
  uint32_t w[2 * sizeof(T)];
};
template <class T>
__device__ __forceinline__ void load_raw(const T* p0, const T* p1, bool vec, Raw<T>& r) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(r.w) = *reinterpret_cast<const uint4*>(p0);
      *reinterpret_cast<uint4*>(r.w + 4) = *reinterpret_cast<const uint4*>(p1);
    } else {
      *reinterpret_cast<uint2*>(r.w) = *reinterpret_cast<const uint2*>(p0);
      *reinterpret_cast<uint2*>(r.w + 2) = *reinterpret_cast<const uint2*>(p1);
    }
  } else {
    T h[8];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = p0[j], h[4 + j] = p1[j];
#pragma unroll
    for (int j = 0; j < int(2 * sizeof(T)); j++) r.w[j] = reinterpret_cast<const uint32_t*>(h)[j];
  }
}
__device__ __forceinline__ void unpack(const Raw<float>& r, float* x) {
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = __uint_as_float(r.w[j]);
}
__device__ __forceinline__ void unpack(const Raw<__half>& r, float* x) {
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = __half2float(__ushort_as_half(uint16_t(r.w[j / 2] >> (16 * (j % 2)))));
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16>& r, float* x) {
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = bits_f(j % 2 ? r.w[j / 2] & 0xffff0000u : r.w[j / 2] << 16);
}
// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// A group of threads has `per` units of one sequence and page, heads one
// after the other, keys before values: the next one's rows come while the
// present one is rounded.
template <int D, int G, class T>
__global__ void __launch_bounds__(256, G == D / 8 ? 4 : 3)
    k_kv8_append(Kv8Args a, Kv8Rows kin, Kv8Rows vin, int blocks, int per, bool vec) {
  constexpr int C = D / 8;                // items a token
  constexpr int N = G == C ? 1 : kItems;  // items a thread
  __shared__ uint32_t red[4 * 8];
  const int tid = threadIdx.x % G;
  const uint32_t group = kv8_append_group(blockIdx.x, threadIdx.x, G);
  const uint32_t parts = (2 * a.heads + per - 1) / per, rest = group / parts;
  const int hb = int(group - rest * parts) * per, he = min(hb + per, 2 * a.heads);
  const int i = min(int(rest / blocks), a.n), b = int(rest % blocks);
  // every thread stays for the exchanges between lanes; `live` ones have work
  bool live = i < a.n;
  Kv8Span sp = {0, 0, 0, false};
  if (live) {
    sp = kv8_span(a, i);
    if (!sp.ok && tid == 0) report(a);
    live = sp.ok;
  }
  const int p0 = sp.len - sp.T;  // below 0: a slot that holds nothing
  const int block = (max(p0, 0) >> a.plog) + b, begin = block << a.plog;
  const int lo = max(p0, begin), hi = min(sp.len, begin + (1 << a.plog));
  live = live && p0 >= 0 && lo < hi;
  if (G > 32 && !live) return;  // a block is one group
  // the page's number comes while the rows do
  const int page = live ? kv8_page(a, i, block) : 0;
  int items = live ? (hi - lo) * C : 0;
  int held = live ? lo - begin : 0;  // tokens that the page holds already

  const auto row_of = [&](int hh) {
    const Kv8Rows& in = hh < a.heads ? kin : vin;
    return static_cast<const T*>(in.p) + int64_t(sp.row + lo - p0) * in.row +
           int64_t(hh < a.heads ? hh : hh - a.heads) * in.head;
  };
  const auto stride_of = [&](int hh) { return hh < a.heads ? kin.row : vin.row; };
  const auto mode_of = [&](int hh) { return hh < a.heads ? a.rope_mode : int(ROPE_NONE); };
  const auto at0 = [&](int mode, int c) { return mode == ROPE_HALVES ? 4 * c : 8 * c; };
  const auto at1 = [&](int mode, int c) { return mode == ROPE_HALVES ? D / 2 + 4 * c : 8 * c + 4; };
  const auto angles = [&](int t, int c) { return a.rope + (int64_t(lo + t) * (D / 2) + 4 * c) * 2; };
  Raw<T> raw[N];
  const auto load = [&](int hh) {
    const T* src = row_of(hh);
    const int64_t st = stride_of(hh);
    const int mode = mode_of(hh);
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int it = tid + u * G, t = it / C, c = it % C;
      if (it < items) load_raw(src + t * st + at0(mode, c), src + t * st + at1(mode, c), vec, raw[u]);
    }
  };
  load(hb);
  if (page < 0) {
    if (live && tid == 0) report(a);
    if (G > 32) return;
    live = false;
    items = held = 0;
  }
  // the unit's largest of numbers that are not negative, as their bits
  // compare (NaN above all). Every lane of a warp is here (a group of fewer
  // than 32 threads has one unit, so its warp's lanes take the same steps). `round` picks the place of its exchange: two for
  // a head and others for the next, since a head may have one exchange alone,
  // and a warp is then past it while another reads
  auto largest = [&](float m, int round) {
    uint32_t v = __float_as_uint(m) & 0x7fffffffu;
    if constexpr (G < 32) {
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(FULL, v, o));
    } else {
      v = __reduce_max_sync(FULL, v);
      if constexpr (G > 32) {
        if (threadIdx.x % 32 == 0) red[8 * round + threadIdx.x / 32] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < G / 32; w++) v = max(v, red[8 * round + w]);
      }
    }
    return __uint_as_float(v);
  };
  for (int hh = hb; hh < he; hh++) {
    const bool key = hh < a.heads;
    const int64_t ph = int64_t(max(page, 0)) * a.heads + (key ? hh : hh - a.heads);
    int8_t* base = (key ? a.k : a.v) + ((ph << a.plog) * D);
    float* sptr = a.scale + 2 * ph + (key ? 0 : 1);
    const float old = held > 0 ? *sptr : 0.f;
    const T* src = row_of(hh);
    const int64_t st = stride_of(hh);
    const int mode = mode_of(hh);
    float y[N][8];
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int it = tid + u * G;
      if (it >= items) continue;
      unpack(raw[u], y[u]);
      if (mode != ROPE_NONE) {
        const float4* cs = reinterpret_cast<const float4*>(angles(it / C, it % C));
        const float4 f0 = cs[0], f1 = cs[1];
        const float co[4] = {f0.x, f0.z, f1.x, f1.z}, si[4] = {f0.y, f0.w, f1.y, f1.w};
        if (mode == ROPE_PAIRS) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float xa = y[u][2 * j], xb = y[u][2 * j + 1];
            y[u][2 * j] = __fmaf_rn(xa, co[j], -__fmul_rn(xb, si[j]));
            y[u][2 * j + 1] = __fmaf_rn(xa, si[j], __fmul_rn(xb, co[j]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float xa = y[u][j], xb = y[u][j + 4];
            y[u][j] = __fmaf_rn(xa, co[j], -__fmul_rn(xb, si[j]));
            y[u][j + 4] = __fmaf_rn(xa, si[j], __fmul_rn(xb, co[j]));
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; j++) most = max_nan(most, fabsf(y[u][j]));
    }
    if (hh + 1 < he) load(hh + 1);
    const int turn = 2 * (hh & 1);
    const float top = largest(most, turn);
    bool slow = !(top < kHuge) || (top > 0.f && top < kTiny);
    float mine = 0.f;  // a/127 as stored, of this thread's candidates
    const float bound = slow ? 0.f : __fmul_rn(top, 1.f - 0x1p-19f);
    if (top != 0.f && (slow || (mode != ROPE_NONE && most >= bound))) {
#pragma unroll
      for (int u = 0; u < N; u++) {
        const int it = tid + u * G;
        uint32_t redo = 0;
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (slow || fabsf(y[u][j]) >= bound) redo |= 1 << j;
        if (it >= items) redo = 0;
        for (; redo; redo &= redo - 1) {
          const int t = it / C, c = it % C;
          const float q = over127(
              value64(src + t * st, at0(mode, c), at1(mode, c), mode, angles(t, c), __ffs(redo) - 1));
          mine = isnan(q) || isnan(mine) ? __int_as_float(0x7fc00000) : fmaxf(mine, q);
        }
      }
    }
    // what is not rotated is exact as it is (and a 32-bit number over 127 is
    // never near the middle of two others: its digits repeat every seven bits)
    const bool exact = mode == ROPE_NONE && !slow;
    float fresh = 0.f;
    // a warp of several units makes the exchange in step, whichever need it
    if (G < 32 || !exact) fresh = largest(mine, turn + 1);
    if (exact) fresh = __fdiv_rn(top, 127.f);
    const float scale = isnan(old) || isnan(fresh) ? __int_as_float(0x7fc00000) : fmaxf(old, fresh);
    const bool some = scale > 0.f;  // not 0, and a number
    slow = slow || scale < kTiny;
    const float back = some ? __fdiv_rn(1.f, scale) : 0.f;
    if (held > 0 && scale > old) {
      const float r = __fmul_rn(old, back);
      uint4* w = reinterpret_cast<uint4*>(base);
      for (int j = tid; j < held * (D / 16); j += G) {
        const uint4 q = w[j];
        w[j] = make_uint4(scaled_bytes(q.x, r, old, scale, slow), scaled_bytes(q.y, r, old, scale, slow),
                          scaled_bytes(q.z, r, old, scale, slow), scaled_bytes(q.w, r, old, scale, slow));
      }
    }
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int it = tid + u * G;
      if (it >= items) continue;
      const int t = it / C, c = it % C;
      float q[8];
      uint32_t redo = slow ? 255 : 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        bool near;
        q[j] = rounded(y[u][j], back, &near);
        if (near) redo |= 1 << j;
      }
      uint2 w = make_uint2(low_bytes(q), low_bytes(q + 4));
      if (!some) w = make_uint2(0, 0), redo = 0;
      for (; redo; redo &= redo - 1) {
        const int j = __ffs(redo) - 1, at = 8 * (j & 3);
        const double x = value64(src + t * st, at0(mode, c), at1(mode, c), mode, angles(t, c), j);
        const uint32_t half = j < 4 ? w.x : w.y;
        const int v = slow ? rounded64(x, scale) : settle(x, double(scale), int8_t(half >> at));
        const uint32_t put = (half & ~(255u << at)) | uint32_t(v & 255) << at;
        if (j < 4)
          w.x = put;
        else
          w.y = put;
      }
      int8_t* dst = base + (held + t) * D;
      if (mode == ROPE_HALVES) {
        *reinterpret_cast<uint32_t*>(dst + 4 * c) = w.x;
        *reinterpret_cast<uint32_t*>(dst + D / 2 + 4 * c) = w.y;
      } else {
        *reinterpret_cast<uint2*>(dst + 8 * c) = w;
      }
    }
    // every thread of the unit has read the old scale: the exchanges above
    // are behind that read
    if (live && tid == 0) *sptr = scale;
  }
}

// --------------------------------------------------------------- read ----
//
// The values of stored tokens: q·scale in 32 bits, rounded once to the
// output's type. A thread has sixteen bytes of outputs of up to kReads
// tokens at a time, neighbours' next to its own: X threads over a token's
// heads, keys and values, 256/X tokens side by side. 12000 tokens, 16 heads
// and sides of 128, bfloat16: 20 us, 3.7 TB/s read and written.
constexpr int kReads = 4;

template <int D, class T>
__global__ void __launch_bounds__(256) k_kv8_read(Kv8Args a, Kv8Rows kout, Kv8Rows vout, int xlog, bool vec) {
  constexpr int V = 16 / sizeof(T), C = D / V;  // values a thread, threads a token and head
  const int i = blockIdx.y;
  const Kv8Span sp = kv8_span(a, i);
  if (!sp.ok) {
    if (threadIdx.x == 0) report(a);
    return;
  }
  const int p0 = sp.len - sp.T, X = 1 << xlog, Y = 256 >> xlog;
  const int t0 = blockIdx.x * (kReads * Y) + (threadIdx.x >> xlog);
  if (p0 < 0 || t0 >= sp.T) return;
  int page[kReads];
#pragma unroll
  for (int u = 0; u < kReads; u++) {
    const int t = t0 + u * Y;
    page[u] = t < sp.T ? kv8_page(a, i, (p0 + t) >> a.plog) : -2;
    if (page[u] == -1) report(a);
  }
  for (int x = threadIdx.x & (X - 1); x < 2 * a.heads * C; x += X) {
    const int hh = x / C, e = x % C * V;
    const bool key = hh < a.heads;
    const int h = key ? hh : hh - a.heads;
    const Kv8Rows& o = key ? kout : vout;
    if (!o.p) continue;
    uint32_t q[kReads][V / 4];
    float s[kReads];
#pragma unroll
    for (int u = 0; u < kReads; u++) {
      const int64_t ph = int64_t(max(page[u], 0)) * a.heads + h;
      const int slot = (p0 + t0 + u * Y) & ((1 << a.plog) - 1);
      const int8_t* from = (key ? a.k : a.v) + ((ph << a.plog) + slot) * D + e;
      s[u] = a.scale[2 * ph + (key ? 0 : 1)];
#pragma unroll
      for (int w = 0; w < V / 4; w++) q[u][w] = reinterpret_cast<const uint32_t*>(from)[w];
    }
    T* dst = static_cast<T*>(const_cast<void*>(o.p)) + int64_t(sp.row + t0) * o.row + int64_t(h) * o.head + e;
#pragma unroll
    for (int u = 0; u < kReads; u++, dst += Y * o.row) {
      if (page[u] < 0) continue;
      __align__(16) T y[V];
#pragma unroll
      for (int j = 0; j < V; j++) narrow(__fmul_rn(float(int8_t(q[u][j / 4] >> (8 * (j % 4)))), s[u]), &y[j]);
      if (vec) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(y);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++) dst[j] = y[j];
      }
    }
  }
}

// One page of one layer a block.
__global__ void __launch_bounds__(256) k_kv8_copy_pages(Kv8Args a, int bytes, const int* from, const int* to) {
  const int f = from[blockIdx.x], t = to[blockIdx.x];
  if (f < 0 || t < 0 || f >= a.pages || t >= a.pages) return;
  const int64_t layer = int64_t(blockIdx.y) * a.pages;
  int8_t* const pool[2] = {a.k + layer * bytes, a.v + layer * bytes};
  for (int j = 0; j < 2; j++) {
    const uint4* src = reinterpret_cast<const uint4*>(pool[j] + int64_t(f) * bytes);
    uint4* dst = reinterpret_cast<uint4*>(pool[j] + int64_t(t) * bytes);
    for (int x = threadIdx.x; x < bytes / 16; x += 256) dst[x] = src[x];
  }
  float* scale = a.scale + layer * a.heads * 2;
  for (int x = threadIdx.x; x < 2 * a.heads; x += 256)
    scale[int64_t(t) * a.heads * 2 + x] = scale[int64_t(f) * a.heads * 2 + x];
}

template <int D, class T>
cudaError_t append_t(const Kv8Args& a, const Kv8Rows& k, const Kv8Rows& v, cudaStream_t st) {
  const int page = 1 << a.plog;
  const int blocks = int(kv8_append_pages(a.max_new, page));
  const int64_t units = int64_t(a.n) * blocks * 2 * a.heads;
  const bool vec = aligned<T>(k, 4) && aligned<T>(v, 4);
  // One token to a sequence: as many threads as hold it. A warp while its
  // registers hold a unit's new values, else eight: 64 tokens of 128 values
  // are kItems items of 256 threads. These take several units in a row where
  // there are blocks enough without.
  int per = 1;
  const auto grid = [&](int g) {
    return kv8_append_grid(int64_t(a.n) * blocks * ((2 * a.heads + per - 1) / per), g);
  };
  if (a.max_new == 1) {
    k_kv8_append<D, D / 8, T><<<grid(D / 8), 256, 0, st>>>(a, k, v, blocks, per, vec);
  } else if (std::min(a.max_new, page) * (D / 8) <= 32 * kItems) {
    k_kv8_append<D, 32, T><<<grid(32), 256, 0, st>>>(a, k, v, blocks, per, vec);
  } else {
    while (per < 2 * a.heads && units >= int64_t(2 * per) * 6 * kSMs) per *= 2;
    k_kv8_append<D, 256, T><<<grid(256), 256, 0, st>>>(a, k, v, blocks, per, vec);
  }
  return cudaGetLastError();
}

template <int D, class T>
cudaError_t read_t(const Kv8Args& a, const Kv8Rows& k, const Kv8Rows& v, cudaStream_t st) {
  const bool vec = (!k.p || aligned<T>(k, 16 / sizeof(T))) && (!v.p || aligned<T>(v, 16 / sizeof(T)));
  int xlog = 4;  // threads over a token
  while (xlog < 8 && 1 << xlog < 2 * a.heads * (D / int(16 / sizeof(T)))) xlog++;
  // no sequence has more tokens than its row of the table has room for, at
  // most 2^31 − 64: the kernel's token numbers stay in 32 bits with any max_new
  const int most = int(std::min<int64_t>(a.max_new, int64_t(a.width) << a.plog)), tokens = kReads * (256 >> xlog);
  k_kv8_read<D, T><<<dim3(unsigned((most - 1) / tokens + 1), a.n), 256, 0, st>>>(a, k, v, xlog, vec);
  return cudaGetLastError();
}

// ------------------------------------------------------------- attend ----
//
// One pass over a sequence's keys and values with the running maximum and
// sum of the softmax, on the tensor cores' integer and half products, with
// sixteen keys as a product's rows and eight queries as its columns.
//
// Scores. A query's values become whole numbers of amax/2^22, written as
// three signed digits in base 256, so the products with the cache's bytes are
// exact integer products (m16n8k32) straight from the bytes as they were
// loaded: no conversion of a key, and 32-bit scores. (Two digits would do
// for 16-bit outputs, not for lse.)
// Values. A byte is exact in float16: below 0x64 its bits ^ 0x80 are the
// number 1024 + 128 + byte, and one subtraction leaves it. The weight is
// w = 2^11·p·s_v/W, with W of each query's own, at least a sixteenth of its
// largest p·s_v so far: a float16 for 16-bit outputs (off by 2^-12 of itself,
// half of what a float16 output is rounded by) and the sum of two for float32
// ones (2^-22), or by 2^-36 W where that is more. So thousands of small
// weights beside a large one are not lost, and pages of large values that a
// query hardly looks at cost it nothing. (With W the largest value scale of
// the sequence and no 2^11 the one lost 2e-3 of the output, 32768 keys 16.6
// nats below another, and the other the ratio of the values in bits.) A query's maximum and W move together, when
// a score passes the one by 2^8 or a weight the other by 2^4.
//
// Layout. A warp takes sixteen tokens at a time from a ring of its own in
// shared memory (Ring, below): a key row's bytes are spread over four lanes,
// sixteen consecutive ones each, a value row's over eight. No block-wide
// synchronisation in the loop: WU warps of a block, and the blocks of a
// cluster, take separate stretches of the keys and are joined at the end
// through (distributed) shared memory; with WU = 1 each warp has a unit of
// its own and writes it out. The references move seldom, so most steps need
// no exchange between lanes.
//
// Bound by the arithmetic of the digits and weights: 48 sequences of 1 to
// 12001 tokens, 4 heads of 128 with 4 queries each, float16: 69 us, 3.4 TB/s
// of the cache. One sequence of 32768 tokens, 8 heads with 4 queries each:
// 33 us, 2.0 TB/s, on the 128 blocks that clusters of 16 give.

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Byte b (0..3) of x and of y as float16s, x's in the low half.
template <int B>
__device__ __forceinline__ uint32_t bytes_f16(uint32_t x, uint32_t y) {
  const uint32_t u = (__byte_perm(x, y, B | (4 + B) << 8) & 0x00ff00ffu) ^ 0x64806480u;
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(u), "r"(0xe480e480u));
  return d;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float at p's place in the shared memory of the cluster's block `rank`.
__device__ __forceinline__ float peer_f32(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
  return v;
}

// Which bytes of a transposed pair of weights the column g takes into word
// n of its operand: `bytes` (two selectors) at the place of the column's
// keys, 0 elsewhere. Keys t = g/2: word t/2, bytes 2·(t % 2).
__device__ __forceinline__ uint32_t column_bytes(int g, int n, uint32_t bytes) {
  const int t = g >> 1;
  if (t >> 1 != n) return 0x4444;
  return t & 1 ? bytes << 8 | 0x44 : 0x4400 | bytes;
}

// Tiles of sixteen tokens come from the cache into a warp's own ring in
// shared memory by 16-byte asynchronous copies: what is under way is bounded
// by shared memory, not by registers (loads straight into the products'
// registers, with one step of 32 tokens ahead, read 5.5 TB/s of long
// sequences and 3.3 of short ones). The chunks of a tile are placed so that
// the products' loads meet no bank twice.
template <int D>
struct Ring {
  static constexpr int half = 16 * D, tile = 2 * half;  // bytes of a tile's keys (or values), and of both
  uint32_t base;                 // the ring
  uint32_t kdst, vdst[2];        // this lane's first chunk of a tile's keys and values (even, odd ones)
  uint32_t ksrc[D / 64], vsrc[2];  // what it reads as operands: of the tokens g, and 2·tg (+ 1)
  const int8_t *k, *v;           // the head's bytes in page 0, at this lane's chunk
  int pbytes, smask;

  __device__ __forceinline__ Ring(const Kv8Args& a, int h, const void* at, int lane) {
    const int g = lane >> 2, tg = lane & 3;
    base = uint32_t(__cvta_generic_to_shared(at));
    const int c = lane % (D / 16), t = lane / (D / 16);  // chunk, token
    if constexpr (D == 64) {
      kdst = 16 * lane;
      vdst[0] = vdst[1] = 64 * (t ^ (t >> 1 & 1)) + 16 * (c ^ (t >> 2 & 1) << 1);
      ksrc[0] = 64 * g + 16 * tg;
#pragma unroll
      for (int r = 0; r < 2; r++)
        vsrc[r] = half + 64 * (2 * tg + (r ^ (tg & 1))) + 16 * (g >> 1 ^ (tg >> 1) << 1) + 8 * (g & 1);
    } else {
      kdst = 128 * t + 16 * (c ^ (t & 1) << 2);
#pragma unroll
      for (int r = 0; r < 2; r++) vdst[r] = 128 * t + 16 * (c ^ (t & 2) ^ r << 2);
#pragma unroll
      for (int j = 0; j < D / 64; j++) ksrc[j] = 128 * g + 16 * (tg + 4 * j ^ (g & 1) << 2);
#pragma unroll
      for (int r = 0; r < 2; r++) vsrc[r] = half + 128 * (2 * tg + r) + 16 * (g ^ 2 * tg);
    }
    k = a.k + ((int64_t(h) << a.plog) * D) + 16 * lane;
    v = a.v + ((int64_t(h) << a.plog) * D) + 16 * lane;
    pbytes = (a.heads << a.plog) * D;  // at most 2^23
    smask = (1 << a.plog) - 1;
  }
  // Tile c of its sequence, of the page `page` (no page: any bytes will do,
  // the tile's keys are hidden), into the ring's place n.
  __device__ __forceinline__ void fetch(int n, int page, int c) const {
    const int64_t off = int64_t(max(page, 0)) * pbytes + ((c << 4) & smask) * D;
    const uint32_t to = base + n * tile;
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kdst + 512 * i), "l"(k + off + 512 * i));
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + half + vdst[i & 1] + 512 * i),
                   "l"(v + off + 512 * i));
    }
  }
  // Sixteen bytes 16·tg .. of each 64 of the keys g and g + 8.
  __device__ __forceinline__ void keys(int n, uint4 (&x)[2][D / 64]) const {
    const uint32_t from = base + n * tile;
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int j = 0; j < D / 64; j++)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[r][j].x), "=r"(x[r][j].y), "=r"(x[r][j].z), "=r"(x[r][j].w)
                     : "r"(from + ksrc[j] + 8 * r * D));
  }
  // Values g·D/8 .. of the tokens 2tg, 2tg + 1, 2tg + 8, 2tg + 9: D/32 words each.
  __device__ __forceinline__ void values(int n, uint32_t (&x)[4][D / 32]) const {
    const uint32_t from = base + n * tile;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t at = from + vsrc[r & 1] + (r >> 1) * 8 * D;
      if constexpr (D == 64)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[r][0]), "=r"(x[r][1]) : "r"(at));
      else
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[r][0]), "=r"(x[r][1]), "=r"(x[r][2]), "=r"(x[r][3])
                     : "r"(at));
    }
  }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The pages of a warp's tiles c0 .. c1 − 1 and their scales: lane l holds
// those of the tile base + l, and the page of the tile base + 32 + l.
struct Pages {
  const Kv8Args& a;
  const float2* scales;
  int i, c1, base, page, ahead;
  float2 scale;

  // `early`: the table's entry of tile `lane`, read before the length was known.
  __device__ __forceinline__ Pages(const Kv8Args& args, int seq, int h, int c0, int c1_, int lane, int early)
      : a(args), scales(reinterpret_cast<const float2*>(args.scale) + h), i(seq), c1(c1_), base(c0) {
    page = c0 == 0 ? (lane < c1 && early >= 0 && early < a.pages ? early : -1) : of(c0 + lane);
    scale = scale_of(page);
    if (page < 0 && c0 + lane < c1) report(a);
    ahead = of(c0 + 32 + lane);
  }
  __device__ __forceinline__ int of(int c) const { return c < c1 ? kv8_page(a, i, c >> (a.plog - 4)) : -1; }
  // No page: 0.
  __device__ __forceinline__ float2 scale_of(int p) const {
    return p < 0 ? make_float2(0.f, 0.f) : sound_scales(scales[int64_t(p) * a.heads]);
  }
  __device__ __forceinline__ void move(int lane) {  // to the next 32 tiles
    base += 32;
    page = ahead;
    if (page < 0 && base + lane < c1) report(a);
    scale = scale_of(page);
    ahead = of(base + 32 + lane);
  }
};
__device__ __forceinline__ int early_page(const Kv8Args& a, int i, int lane) {
  const int b = lane >> (a.plog - 4);
  return b < a.width ? a.table[int64_t(i) * a.width + b] : -1;
}

// Warps of a block, tiles of a warp's ring, blocks that an SM shall hold: by
// registers and by the rings (about 200 KB an SM).
template <int D, int NQ, int WU>
struct Shape {
  static constexpr int warps = WU == 1 ? 4 : WU;
  static constexpr int ring = D == 64 ? 5 : 4;
  static constexpr int blocks = NQ > 1 || WU > 4 ? 2 : D == 64 ? 4 : 3;
  static constexpr size_t digits = size_t(NQ) * 3 * (D / 64) * 32 * 16;  // bytes, a unit's
  static constexpr size_t rings = size_t(warps) * ring * Ring<D>::tile;
  // the joined outputs take the rings' place
  static constexpr size_t join = WU == 1 ? 0 : size_t(warps + 1) * 8 * NQ * (D + 2) * 4;
  static constexpr size_t smem = (WU == 1 ? warps : 1) * (digits + size_t(8 * NQ) * 8) + (rings > join ? rings : join);
};

// NP: float16s of a weight.
template <int D, int NQ, int NP, int WU>
__global__ void __launch_bounds__(32 * Shape<D, NQ, WU>::warps, Shape<D, NQ, WU>::blocks)
    k_kv8_attend(Kv8Args a, Kv8Attend t, int type, int S, int qtiles, int units, bool vec, bool ovec) {
  using Sh = Shape<D, NQ, WU>;
  constexpr int NR = 8 * NQ, H2 = D / 64, R = Sh::ring;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
  constexpr int kUnits = WU == 1 ? Sh::warps : 1;
  uint8_t* rings = smem + kUnits * (Sh::digits + NR * 8);
  uint8_t* mine = smem + (WU == 1 ? warp * (Sh::digits + NR * 8) : 0);
  uint4* qd = reinterpret_cast<uint4*>(mine);               // [NQ][3][H2][32]
  float* qf = reinterpret_cast<float*>(mine + Sh::digits);  // [NR]
  int* qpos = reinterpret_cast<int*>(qf + NR);              // [NR]
  float* wm = reinterpret_cast<float*>(rings);              // [WU][NR], WU > 1, when the rings are done
  float* wl = wm + WU * NR;
  float* wo = wl + WU * NR;                                 // [WU][NR][D]
  float* bm = wo + WU * NR * D;                             // [NR], [NR], [NR][D]
  float* bl = bm + NR;
  float* bo = bl + NR;

  const int rank = S > 1 ? int(cluster_rank()) : 0;
  const int unit = WU == 1 ? blockIdx.x * Sh::warps + warp : blockIdx.x / S;
  if (unit >= units) return;
  const int h = unit % a.heads, qt = unit / a.heads % qtiles, i = unit / a.heads / qtiles;
  const int group = t.heads / a.heads;
  const int early = early_page(a, i, lane);
  const Kv8Span sp = kv8_span(a, i);
  if (!sp.ok) {
    if ((WU == 1 ? lane : tid) == 0) report(a);
    return;  // every block of the cluster: it has one sequence
  }
  const int r0 = qt * NR, nrow = min(NR, sp.T * group - r0);  // this unit's query rows
  if (nrow <= 0) return;
  const int p0 = sp.len - sp.T;
  const int pmin = p0 + r0 / group, pmax = p0 + (r0 + nrow - 1) / group;
  const int first = a.first ? max(0, a.first[i]) : 0;
  const int klo = max(first, t.window > 0 ? pmin - t.window + 1 : 0), khi = pmax + 1;
  const int cb = klo >> 4, ce = max(cb, (khi + 15) >> 4);
  const int per = (ce - cb + S * WU - 1) / (S * WU);
  const int c0 = min(ce, cb + (WU == 1 ? 0 : rank * WU + warp) * per), c1 = min(ce, c0 + per);

  Pages pages(a, i, h, c0, c1, lane, early);
  const Ring<D> ring(a, h, rings + warp * R * Ring<D>::tile, lane);
  // tiles are fetched in order, R − 1 ahead of the one in use, a group of copies each
  int fc = c0;
  auto fetch = [&](int n, int page) {
    if (fc < c1) ring.fetch(n, page, fc);
    copies_commit();
    fc++;
  };
#pragma unroll
  for (int u = 0; u < R - 1; u++) fetch(u, __shfl_sync(FULL, pages.page, u));

  // --- the queries: rotated, and written as digits ---
  for (int nq = WU == 1 ? 0 : warp; nq < NQ; nq += WU) {
    const int r = nq * 8 + g;  // this lane's query
    const bool there = r < nrow;
    const int tq = there ? (r0 + r) / group : 0, hq = h * group + (there ? (r0 + r) % group : 0);
    const int pos = p0 + tq;
    float x[H2][16];
    const int64_t off = int64_t(sp.row + tq) * t.q.row + int64_t(hq) * t.q.head + 16 * tg;
    load_row<D>(t.q.p, off, type, vec, there, x);
    rotate16<D>(x, a, pos, tg);
    const float amax = group_amax<D>(x, FULL);  // NaN where a value is none
    const float to = lift_row<D>(x, amax);
#pragma unroll
    for (int j = 0; j < H2; j++) {
      uint32_t y[16];
#pragma unroll
      for (int e = 0; e < 16; e++) y[e] = digits_of(__fmaf_rn(x[j][e], to, MAGIC));
#pragma unroll
      for (int d = 0; d < 3; d++)
        qd[((nq * 3 + d) * H2 + j) * 32 + lane] =
            make_uint4(take_bytes(y, d), take_bytes(y + 4, d), take_bytes(y + 8, d), take_bytes(y + 12, d));
    }
    if (tg == 0) {
      // scores in units of log 2; a query that is no number has no score
      qf[r] = __fmul_rn(__fmul_rn(amax, 1.f / kQueryUnits), __fmul_rn(t.scale, 1.44269504f));
      qpos[r] = there ? pos : -1;
    }
  }
  if (WU == 1)
    __syncwarp();
  else
    __syncthreads();

  // --- the pass over the keys ---
  float o[NQ][D / 16][4] = {};
  // a query's largest score (about), sum, score factor, 2^11/W, and log2 of 2^4·W
  float ref[NQ][2], l[NQ][2] = {}, f[NQ][2], toW[NQ][2], most[NQ][2];
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      ref[nq][j] = ninf();
      toW[nq][j] = pow2(253);
      most[nq][j] = ninf();
      f[nq][j] = qf[nq * 8 + 2 * tg + j];
    }
  // tiles that every query of the unit sees whole
  const int in_lo = max(first, t.window > 0 ? pmax - t.window + 1 : 0), in_hi = pmin;
  auto step = [&](int n, int c) {
    const int j = c - pages.base;
    const int page = __shfl_sync(FULL, pages.page, j);
    const float bsk = __shfl_sync(FULL, pages.scale.x, j), bsv = __shfl_sync(FULL, pages.scale.y, j);
    const bool edge = page < 0 || c * 16 < in_lo || c * 16 + 15 > in_hi;
    uint4 bk[2][H2];
    ring.keys(n, bk);
    uint32_t pw[NQ][NP][2];  // the weights, transposed: queries in rows
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
      int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
      auto digit = [&](int* acc, int d) {
#pragma unroll
        for (int j = 0; j < H2; j++) {
          const uint4 q = qd[((nq * 3 + d) * H2 + j) * 32 + lane];
          mma_s8(acc, bk[0][j].x, bk[1][j].x, bk[0][j].y, bk[1][j].y, q.x, q.y);
          mma_s8(acc, bk[0][j].z, bk[1][j].z, bk[0][j].w, bk[1][j].w, q.z, q.w);
        }
      };
      // the two upper digits share an accumulator: 128·128·16512 < 2^31
      digit(hi, 2);
#pragma unroll
      for (int j = 0; j < 4; j++) hi[j] <<= 8;
      digit(hi, 1);
      digit(lo, 0);
      float s[4], x[4];
      const float fs[2] = {__fmul_rn(f[nq][0], bsk), __fmul_rn(f[nq][1], bsk)};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        s[j] = __fmaf_rn(256.f, float(hi[j]), float(lo[j]));
        x[j] = __fmaf_rn(s[j], fs[j & 1], -ref[nq][j & 1]);
      }
      bool hide[4] = {false, false, false, false};
      if (edge) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int p = qpos[nq * 8 + 2 * tg + (j & 1)], key = c * 16 + g + (j >> 1) * 8;
          hide[j] = key > p || key < first || (t.window > 0 && key <= p - t.window) || page < 0;
          if (hide[j]) x[j] = ninf();
        }
      }
      // (A scale far above W has a term of 0, or as far below 1: no infinity
      // here, and none for what is hidden, whose term is 0 whatever its page's
      // scale. Where that is no number, the terms of what is seen are none.)
      float sv[2];
#pragma unroll
      for (int j = 0; j < 2; j++) sv[j] = fminf(__fmul_rn(bsv, toW[nq][j]), 3.4e38f);
      const float heavy = lg2(bsv);
      // before its first key a query's reference is −inf, and any score above
      if (__any_sync(FULL, fmaxf(x[0], x[2]) > fminf(8.f, __fsub_rn(most[nq][0], heavy)) ||
                               fmaxf(x[1], x[3]) > fminf(8.f, __fsub_rn(most[nq][1], heavy)))) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float m = fmaxf(hide[j] ? ninf() : __fmul_rn(s[j], fs[j]), hide[j + 2] ? ninf() : __fmul_rn(s[j + 2], fs[j]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
          m = fmaxf(m, ref[nq][j]);
          const float r = ref[nq][j] == m ? 1.f : ex2(__fsub_rn(ref[nq][j], m));
          ref[nq][j] = m;
          l[nq][j] = __fmul_rn(l[nq][j], r);
          x[j] = hide[j] ? ninf() : __fmaf_rn(s[j], fs[j], -m);
          x[j + 2] = hide[j + 2] ? ninf() : __fmaf_rn(s[j + 2], fs[j], -m);
          // the largest weight, hidden keys' of an unsound scale aside
          float u = fmaxf(__fmul_rn(ex2(x[j]), bsv), __fmul_rn(ex2(x[j + 2]), bsv));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) u = fmaxf(u, __shfl_xor_sync(FULL, u, d));
          const float unit = __fmul_rn(inverse<NP>(toW[nq][j]), r);  // what o's unit, 2^-11 W, is worth now
          toW[nq][j] = weight_scale<NP>(fmaxf(u, __fmul_rn(unit, 2048.f)), &most[nq][j]);
          sv[j] = fminf(__fmul_rn(bsv, toW[nq][j]), 3.4e38f);
          const float k = __fmul_rn(unit, toW[nq][j]);
#pragma unroll
          for (int mt = 0; mt < D / 16; mt++) {
            o[nq][mt][j] = __fmul_rn(o[nq][mt][j], k);
            o[nq][mt][j + 2] = __fmul_rn(o[nq][mt][j + 2], k);
          }
        }
      }
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float p = ex2(x[j]);
        l[nq][j & 1] = __fadd_rn(l[nq][j & 1], p);
        w[j] = __fmul_rn(p, sv[j & 1]);
      }
#pragma unroll
      for (int n = 0; n < NP; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint32_t y = pack_f16(w[2 * j], w[2 * j + 1]);
          if (n + 1 < NP) {
            w[2 * j] = __fsub_rn(w[2 * j], __half2float(__ushort_as_half(y & 0xffff)));
            w[2 * j + 1] = __fsub_rn(w[2 * j + 1], __half2float(__ushort_as_half(y >> 16)));
          }
          pw[nq][n][j] = transpose8(y);
        }
    }
    uint32_t bv[4][D / 32];
    ring.values(n, bv);
    auto values = [&](auto MT) {
      constexpr int mt = decltype(MT)::value, wd = mt / 2, by = 2 * (mt % 2);
      const uint32_t a0 = bytes_f16<by>(bv[0][wd], bv[1][wd]), a1 = bytes_f16<by + 1>(bv[0][wd], bv[1][wd]);
      const uint32_t a2 = bytes_f16<by>(bv[2][wd], bv[3][wd]), a3 = bytes_f16<by + 1>(bv[2][wd], bv[3][wd]);
#pragma unroll
      for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int n = 0; n < NP; n++) mma_f16(o[nq][mt], a0, a1, a2, a3, pw[nq][n][0], pw[nq][n][1]);
    };
    values(std::integral_constant<int, 0>());
    values(std::integral_constant<int, 1>());
    values(std::integral_constant<int, 2>());
    values(std::integral_constant<int, 3>());
    if constexpr (D == 128) {
      values(std::integral_constant<int, 4>());
      values(std::integral_constant<int, 5>());
      values(std::integral_constant<int, 6>());
      values(std::integral_constant<int, 7>());
    }
  };
  int n = 0;
  for (int c = c0; c < c1; c++) {
    if (c - pages.base == 32) pages.move(lane);
    copies_wait<R - 2>();
    __syncwarp();  // every lane's copies of this tile, and its reads of the one before
    {
      // the tile R − 1 further on, into the place that the last step left;
      // its page may be among the next 32 tiles'
      const int j = fc - pages.base, pn = __shfl_sync(FULL, j < 32 ? pages.page : pages.ahead, j & 31);
      fetch(n == 0 ? R - 1 : n - 1, pn);
    }
    step(n, c);
    n = n + 1 == R ? 0 : n + 1;
  }
  if (WU > 1) {
    copies_wait<0>();
    __syncthreads();  // the rings are done: their place is used again
  }
#pragma unroll
  for (int nq = 0; nq < NQ; nq++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[nq][j] = __fadd_rn(l[nq][j], __shfl_xor_sync(FULL, l[nq][j], d));

  if constexpr (WU == 1) {
    // a lane's D/8 values of two queries, straight out
    constexpr int E = D / 8;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int r = nq * 8 + 2 * tg + j;
        const bool there = r < nrow;
        const int tq = there ? (r0 + r) / group : 0, hq = h * group + (there ? (r0 + r) % group : 0);
        const float inv = l[nq][j] == 0.f ? 0.f : __fdiv_rn(inverse<NP>(toW[nq][j]), l[nq][j]);
        float y[E];
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++) {
          y[2 * mt] = __fmul_rn(o[nq][mt][j], inv);
          y[2 * mt + 1] = __fmul_rn(o[nq][mt][j + 2], inv);
        }
        if (t.q8) {
          // blocks of 32 values: over 32/E of the eight lanes of a query
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < E; e++) m = fmaxf(m, fabsf(y[e]));
#pragma unroll
          for (int d = 4; d < 4 * 32 / E; d <<= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
          if (there) {
            const int64_t at = (int64_t(sp.row + tq) * t.heads + hq) * D + g * E;
#pragma unroll
            for (int e = 0; e < E; e += 4) {
              char4 c4;
              c4.x = quant_val(y[e], m), c4.y = quant_val(y[e + 1], m);
              c4.z = quant_val(y[e + 2], m), c4.w = quant_val(y[e + 3], m);
              *reinterpret_cast<char4*>(t.q8 + at + e) = c4;
            }
            if (g * E % 32 == 0) t.q8s[at / QK] = make_float2(quant_scale(m), quant_scale(m));
          }
        }
        if (!there) continue;
        if (t.out.p) {
          const int64_t at = int64_t(sp.row + tq) * t.out.row + int64_t(hq) * t.out.head + g * E;
          if (ovec && type == 0) {
            float4* op = reinterpret_cast<float4*>(static_cast<float*>(const_cast<void*>(t.out.p)) + at);
#pragma unroll
            for (int e = 0; e < E; e += 4) op[e / 4] = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
          } else if (ovec) {
            uint16_t hy[E];
#pragma unroll
            for (int e = 0; e < E; e++)
              hy[e] = type == 1 ? __half_as_ushort(__float2half_rn(y[e]))
                                : __bfloat16_as_ushort(__float2bfloat16_rn(y[e]));
            uint4* op = reinterpret_cast<uint4*>(static_cast<uint16_t*>(const_cast<void*>(t.out.p)) + at);
#pragma unroll
            for (int e = 0; e < E; e += 8)
              op[e / 8] = make_uint4(hy[e] | hy[e + 1] << 16, hy[e + 2] | hy[e + 3] << 16, hy[e + 4] | hy[e + 5] << 16,
                                     hy[e + 6] | hy[e + 7] << 16);
          } else {
#pragma unroll
            for (int e = 0; e < E; e++) put(t, type, at + e, y[e]);
          }
        }
        if (t.lse && g == 0) t.lse[int64_t(sp.row + tq) * t.heads + hq] = lse_of(ref[nq][j], l[nq][j]);
      }
  } else {
    // --- the warps' shares joined ---
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int r = nq * 8 + 2 * tg + j;
        if (r >= nrow) continue;
        if (g == 0) {
          wm[warp * NR + r] = ref[nq][j];
          wl[warp * NR + r] = l[nq][j];
        }
        float* dst = wo + (warp * NR + r) * D + g * (D / 8);
        const float unit = inverse<NP>(toW[nq][j]);
#pragma unroll
        for (int mt = 0; mt < D / 16; mt++)
          *reinterpret_cast<float2*>(dst + 2 * mt) =
              make_float2(__fmul_rn(o[nq][mt][j], unit), __fmul_rn(o[nq][mt][j + 2], unit));
      }
    __syncthreads();
    // Item: 32 values of one row, a lane each. The weight of a share is
    // 2^(its reference − the largest); one without keys counts 0 (its
    // reference is −inf), and where all are, the sums are 0 or no number.
    auto weight = [](float mi, float top) { return mi == top ? 1.f : ex2(__fsub_rn(mi, top)); };
    auto finish = [&](int r, int d, float top, float sum, float val) {
      const int tq = (r0 + r) / group, hq = h * group + (r0 + r) % group;
      const float y = sum == 0.f ? 0.f : __fdiv_rn(val, sum);
      if (t.out.p) put(t, type, int64_t(sp.row + tq) * t.out.row + int64_t(hq) * t.out.head + d, y);
      if (t.q8) {
        const int64_t at = int64_t(sp.row + tq) * t.heads * D + hq * D + d;
        float s;
        t.q8[at] = quant_lane(y, &s);
        if (lane == 0) t.q8s[at / QK] = make_float2(s, s);
      }
      if (t.lse && d == 0) t.lse[int64_t(sp.row + tq) * t.heads + hq] = lse_of(top, sum);
    };
    const int items = nrow * (D / 32);
    for (int it = warp; it < items; it += WU) {
      const int r = it / (D / 32), d = it % (D / 32) * 32 + lane;
      float top = wm[r], sum = 0.f, val = 0.f;
#pragma unroll
      for (int w = 1; w < WU; w++) top = fmaxf(top, wm[w * NR + r]);
#pragma unroll
      for (int w = 0; w < WU; w++) {
        const float k = weight(wm[w * NR + r], top);
        sum = __fmaf_rn(k, wl[w * NR + r], sum);
        val = __fmaf_rn(k, wo[(w * NR + r) * D + d], val);
      }
      if (S == 1) {
        finish(r, d, top, sum, val);
      } else {
        bo[r * D + d] = val;
        if (d == 0) {
          bm[r] = top;
          bl[r] = sum;
        }
      }
    }
    if (S == 1) return;
    cluster_sync();
    for (int it = rank * WU + warp; it < items; it += S * WU) {
      const int r = it / (D / 32), d = it % (D / 32) * 32 + lane;
      float top = ninf(), sum = 0.f, val = 0.f;
      for (int b = 0; b < S; b++) top = fmaxf(top, peer_f32(bm + r, b));
      for (int b = 0; b < S; b++) {
        const float k = weight(peer_f32(bm + r, b), top);
        sum = __fmaf_rn(k, peer_f32(bl + r, b), sum);
        val = __fmaf_rn(k, peer_f32(bo + r * D + d, b), val);
      }
      finish(r, d, top, sum, val);
    }
    cluster_sync();  // no block leaves while another reads its shared memory
  }
}

// ---------------------------------------------- attend, one query a head ----
//
// Where a sequence's key head has one query (a single token, as many query
// heads as key heads: the flow LM's step), seven of a product's eight
// columns would be empty. Here they hold the digits instead, and a warp
// takes 32 tokens at a time:
//  * the query's digits stand in the columns (the lowest in even ones, the
//    middle in odd ones, the highest added to odd ones), so every lane has
//    the digits of four keys and takes one of them: one score, one
//    exponential and one weight a lane for 32 keys;
//  * the weight, a key's softmax term times its page's value scale, is a
//    whole number of 2^-32 of a reference W, a power of two above the largest
//    such product so far and at most twice it; one 8x8 transposition brings
//    its four bytes for all 32 keys to the columns of integer products with
//    the values' bytes (m16n8k32, unsigned weights): the four keys of a row
//    group in columns of their own, the bytes 0 and 2 in one product, 1 and 3
//    in another. So a weight has all of a float's bits down to 2^-8 of W, and
//    below that it is off by 2^-33 W at most: thousands of small ones beside a large one are not
//    lost (whole numbers of 2^-23 of the largest value scale lost them, and
//    what stood beside pages of large values that the query did not look at);
//  * the values' bytes need a 4x4 byte transposition (eight byte
//    permutations for sixteen bytes) and no conversion.
// Sums are exact integers until the references move (a larger score, a larger
// weight) or 32768 keys have gone by; then they go into float32 sums. 256
// sequences of 65 to 576 tokens, 16 heads of 64: 38 us, 4.5 TB/s of the cache;
// as many of 8192 tokens 623 us, 6.9 TB/s, and 64 of 16384 336 us, 6.4 TB/s.
__device__ __forceinline__ void mma_s8u8(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Steps of a warp's ring and warps an SM shall hold, by shared memory: heads
// of 64 took 1 to 3 % longer with 2 steps and 16 or 20 warps and with 4 steps
// and 12.
template <int D, int WU>
struct Shape1 {
  static constexpr int warps = WU == 1 ? 4 : WU;
  static constexpr int ring = D == 64 ? 3 : 2;  // steps of 32 tokens
  static constexpr int per_sm = D == 64 ? 16 : 12;  // warps, by registers and rings
  static constexpr int blocks = per_sm / warps < 1 ? 1 : per_sm / warps;
  static constexpr size_t rings = size_t(warps) * ring * 2 * Ring<D>::tile;
  static constexpr size_t smem = rings;  // the joined outputs, smaller, take their place
};

template <int D, int WU>
__global__ void __launch_bounds__(32 * Shape1<D, WU>::warps, Shape1<D, WU>::blocks)
    k_kv8_attend1(Kv8Args a, Kv8Attend t, int type, int S, int units, bool vec) {
  constexpr int H2 = D / 64, M = D / 16, WV = D / 32, R = Shape1<D, WU>::ring;
  constexpr float kOne = 4294967296.f;  // of a weight of W; just below it at most
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);  // [WU][D + 2], and the block's, when the rings are done
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
  const int rank = S > 1 ? int(cluster_rank()) : 0;
  const int unit = WU == 1 ? blockIdx.x * Shape1<D, WU>::warps + warp : blockIdx.x / S;
  if (unit >= units) return;
  const int h = unit % a.heads, i = unit / a.heads;
  const int early = early_page(a, i, lane);
  const Kv8Span sp = kv8_span(a, i);
  if (!sp.ok) {
    if ((WU == 1 ? lane : tid) == 0) report(a);
    return;
  }
  if (sp.T == 0) return;
  const int p = sp.len - 1;  // the query's position
  const int first = max(a.first ? max(0, a.first[i]) : 0, t.window > 0 ? p - t.window + 1 : 0);
  const int cb = first >> 4, ce = max(cb, (p + 16) >> 4);
  const int per = ((ce - cb + S * WU - 1) / (S * WU) + 1) & ~1;  // whole steps
  const int c0 = min(ce, cb + (WU == 1 ? 0 : rank * WU + warp) * per), c1 = min(ce, c0 + per);

  Pages pages(a, i, h, c0, c1, lane, early);
  const Ring<D> ring(a, h, smem + warp * R * 2 * Ring<D>::tile, lane);
  // steps of two tiles are fetched in order, R − 1 ahead of the one in use, a group of copies each
  int fc = c0;
  auto fetch = [&](int n, int pa, int pb) {
    if (fc < c1) {
      ring.fetch(2 * n, pa, fc);
      ring.fetch(2 * n + 1, pb, fc + 1);
    }
    copies_commit();
    fc += 2;
  };
#pragma unroll
  for (int u = 0; u < R - 1; u++)
    fetch(u, __shfl_sync(FULL, pages.page, 2 * u), __shfl_sync(FULL, pages.page, 2 * u + 1));

  // --- the query: rotated, and written as digits ---
  uint32_t q01[H2][4], q2[H2][4];
  float f;
  {
    float x[H2][16];
    const int64_t off = int64_t(sp.row) * t.q.row + int64_t(h) * t.q.head + 16 * tg;
    load_row<D>(t.q.p, off, type, vec, true, x);
    rotate16<D>(x, a, p, tg);
    const float amax = group_amax<D>(x, FULL);  // NaN where a value is none
    const float to = lift_row<D>(x, amax);
#pragma unroll
    for (int j = 0; j < H2; j++)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        uint32_t n[4];
#pragma unroll
        for (int e = 0; e < 4; e++) n[e] = digits_of(__fmaf_rn(x[j][4 * w + e], to, MAGIC));
        q01[j][w] = take_bytes(n, g & 1);
        q2[j][w] = g & 1 ? take_bytes(n, 2) : 0;
      }
    f = __fmul_rn(__fmul_rn(amax, 1.f / kQueryUnits), __fmul_rn(t.scale, 1.44269504f));
  }

  // --- the pass over the keys: lane (g, tg) has key g + 8·(tg & 1) of tile tg >> 1 ---
  const uint32_t at0 = column_bytes(g, 0, 0x20), at1 = column_bytes(g, 1, 0x20);
  const uint32_t odd0 = column_bytes(g, 0, 0x31), odd1 = column_bytes(g, 1, 0x31);
  int ev[M][4] = {}, od[M][4] = {};  // sums over the weights' bytes 0 (even columns) and 2 (odd), 1 and 3
  float o[M][2] = {};
  float ref = ninf(), l = 0.f, W = pow2(12), toW = pow2(242), most = ninf();  // 1/W; log2 of W
  int held = 0;  // steps in the integer sums
  // the integer sums into the float ones, and these times r
  auto flush = [&](float r) {
#pragma unroll
    for (int mt = 0; mt < M; mt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float lo = __fmaf_rn(256.f, float(od[mt][2 * e]), float(ev[mt][2 * e]));
        const float hi = __fmaf_rn(256.f, float(od[mt][2 * e + 1]), float(ev[mt][2 * e + 1]));
        o[mt][e] = __fmul_rn(r, __fadd_rn(o[mt][e], __fmaf_rn(65536.f, hi, lo)));
        ev[mt][2 * e] = ev[mt][2 * e + 1] = od[mt][2 * e] = od[mt][2 * e + 1] = 0;
      }
    held = 0;
  };
  auto step = [&](int n, int c) {
    const int j = c - pages.base;
    const int pa = __shfl_sync(FULL, pages.page, j), pb = __shfl_sync(FULL, pages.page, j + 1);
    const float sva = __shfl_sync(FULL, pages.scale.y, j), svb = __shfl_sync(FULL, pages.scale.y, j + 1);
    const float fs = __fmul_rn(f, __shfl_sync(FULL, pages.scale.x, j + (tg >> 1)));
    float sv = tg < 2 ? sva : svb;
    const bool edge = (pa | pb) < 0 || c * 16 < first || c * 16 + 31 > p;
    // the highest digit's sums, then the lower ones' on top: even columns
    // the lowest digit, odd ones 256·highest + middle (below 2^31)
    uint4 ka[2][H2], kb[2][H2];
    ring.keys(2 * n, ka);
    ring.keys(2 * n + 1, kb);
    int s0[4] = {0, 0, 0, 0}, s1[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < H2; e++) {
      mma_s8(s0, ka[0][e].x, ka[1][e].x, ka[0][e].y, ka[1][e].y, q2[e][0], q2[e][1]);
      mma_s8(s1, kb[0][e].x, kb[1][e].x, kb[0][e].y, kb[1][e].y, q2[e][0], q2[e][1]);
      mma_s8(s0, ka[0][e].z, ka[1][e].z, ka[0][e].w, ka[1][e].w, q2[e][2], q2[e][3]);
      mma_s8(s1, kb[0][e].z, kb[1][e].z, kb[0][e].w, kb[1][e].w, q2[e][2], q2[e][3]);
    }
    s0[1] <<= 8, s0[3] <<= 8, s1[1] <<= 8, s1[3] <<= 8;
#pragma unroll
    for (int e = 0; e < H2; e++) {
      mma_s8(s0, ka[0][e].x, ka[1][e].x, ka[0][e].y, ka[1][e].y, q01[e][0], q01[e][1]);
      mma_s8(s1, kb[0][e].x, kb[1][e].x, kb[0][e].y, kb[1][e].y, q01[e][0], q01[e][1]);
      mma_s8(s0, ka[0][e].z, ka[1][e].z, ka[0][e].w, ka[1][e].w, q01[e][2], q01[e][3]);
      mma_s8(s1, kb[0][e].z, kb[1][e].z, kb[0][e].w, kb[1][e].w, q01[e][2], q01[e][3]);
    }
    const int lo = tg & 2 ? (tg & 1 ? s1[2] : s1[0]) : (tg & 1 ? s0[2] : s0[0]);
    const int up = tg & 2 ? (tg & 1 ? s1[3] : s1[1]) : (tg & 1 ? s0[3] : s0[1]);
    const float s = __fmaf_rn(256.f, float(up), float(lo));
    float x = __fmaf_rn(s, fs, -ref);
    bool hide = false;
    if (edge) {
      const int key = (c + (tg >> 1)) * 16 + g + 8 * (tg & 1);
      hide = key > p || key < first || (tg < 2 ? pa : pb) < 0;
      if (hide) x = ninf(), sv = 0.f;
    }
    // The references move: a larger score, or a larger weight.
    if (__any_sync(FULL, x > fminf(0.f, __fsub_rn(most, lg2(sv))))) {
      float m = hide ? ninf() : __fmul_rn(s, fs);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
      m = fmaxf(m, ref);
      const float r = ref == m ? 1.f : ex2(__fsub_rn(ref, m));
      ref = m;
      l = __fmul_rn(l, r);
      W = __fmul_rn(W, r);
      x = hide ? ninf() : __fmaf_rn(s, fs, -m);
      float u = __fmul_rn(ex2(x), sv);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) u = fmaxf(u, __shfl_xor_sync(FULL, u, d));
      // the power of two above the largest weight, or what W is worth now
      const int e = unit_of(fmaxf(__fadd_rn(u, u), W));
      toW = pow2(254 - e);
      flush(__fmul_rn(W, toW));
      W = pow2(e);
      most = float(e - 127);
    }
    const float w = x > 0.f ? 1.f : ex2(x);  // above 0 by the rounding of the reference
    l = __fadd_rn(l, w);
    // a scale far above W has a term of 0, or as far below 1: no infinity here
    const uint32_t y = __float2uint_rn(__fmul_rn(__fmul_rn(w, fminf(__fmul_rn(sv, toW), 3.4e38f)), kOne));
    const uint32_t yt = transpose8(y);
    const uint32_t b0 = __byte_perm(yt, 0, at0), b1 = __byte_perm(yt, 0, at1);
    const uint32_t m0 = __byte_perm(yt, 0, odd0), m1 = __byte_perm(yt, 0, odd1);
    uint32_t v[2][4][WV];
    ring.values(2 * n, v[0]);
    ring.values(2 * n + 1, v[1]);
#pragma unroll
    for (int wd = 0; wd < WV; wd++) {
      // four tokens' words of four values each → four words of a value each
      uint32_t d[2][4];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        const uint32_t l01 = __byte_perm(v[m][0][wd], v[m][1][wd], 0x5140),
                       h01 = __byte_perm(v[m][0][wd], v[m][1][wd], 0x7362);
        const uint32_t l23 = __byte_perm(v[m][2][wd], v[m][3][wd], 0x5140),
                       h23 = __byte_perm(v[m][2][wd], v[m][3][wd], 0x7362);
        d[m][0] = __byte_perm(l01, l23, 0x5410);
        d[m][1] = __byte_perm(l01, l23, 0x7632);
        d[m][2] = __byte_perm(h01, h23, 0x5410);
        d[m][3] = __byte_perm(h01, h23, 0x7632);
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const uint32_t av[4] = {d[0][2 * e], d[0][2 * e + 1], d[1][2 * e], d[1][2 * e + 1]};
        mma_s8u8(ev[2 * wd + e], av, b0, b1);
        mma_s8u8(od[2 * wd + e], av, m0, m1);
      }
    }
    if (++held == 1024) flush(1.f);  // 32768 keys: 255·128·32768 < 2^31
  };
  int n = 0;
  for (int c = c0; c < c1; c += 2) {
    if (c - pages.base == 32) pages.move(lane);
    copies_wait<R - 2>();
    __syncwarp();  // every lane's copies of this step, and its reads of the one before
    {
      // the step R − 1 further on, into the place that the last one left; its
      // pages may be among the next 32 tiles'
      const int j = fc - pages.base, from = j < 32 ? pages.page : pages.ahead;
      const int pa = __shfl_sync(FULL, from, j & 31), pb = __shfl_sync(FULL, from, (j & 31) + 1);
      fetch(n == 0 ? R - 1 : n - 1, pa, pb);
    }
    step(n, c);
    n = n + 1 == R ? 0 : n + 1;
  }
  if (WU > 1) {
    copies_wait<0>();
    __syncthreads();  // the rings are done: their place is used again
  }
  flush(1.f);
  // sums over the columns (the lanes of a row group), and over all lanes
#pragma unroll
  for (int mt = 0; mt < M; mt++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      o[mt][e] = __fadd_rn(o[mt][e], __shfl_xor_sync(FULL, o[mt][e], 1));
      o[mt][e] = __fadd_rn(o[mt][e], __shfl_xor_sync(FULL, o[mt][e], 2));
    }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) l = __fadd_rn(l, __shfl_xor_sync(FULL, l, d));

  // lane (g, tg) goes on with D/32 of row group g's D/8 values
  constexpr int E = D / 32;
  float y[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    float v = o[e / 2][e % 2];
#pragma unroll
    for (int n = 1; n < 4; n++)
      if (tg == n) v = o[(n * E + e) / 2][e % 2];
    y[e] = __fmul_rn(__fmul_rn(v, 1.f / kOne), W);  // W is 0 where there was no key
  }
  const int d0 = g * (D / 8) + tg * E;
  auto finish = [&](float top, float sum, const float* val) {
    float r[E], m = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      r[e] = sum == 0.f ? 0.f : __fdiv_rn(val[e], sum);
      m = fmaxf(m, fabsf(r[e]));
    }
    if (t.out.p) {
      const int64_t at = int64_t(sp.row) * t.out.row + int64_t(h) * t.out.head + d0;
#pragma unroll
      for (int e = 0; e < E; e++) put(t, type, at + e, r[e]);
    }
    if (t.q8) {  // blocks of 32 values: 32/E lanes
#pragma unroll
      for (int d = 1; d < 32 / E; d <<= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, d));
      const int64_t at = (int64_t(sp.row) * t.heads + h) * D + d0;
#pragma unroll
      for (int e = 0; e < E; e++) t.q8[at + e] = quant_val(r[e], m);
      if (d0 % QK == 0) t.q8s[at / QK] = make_float2(quant_scale(m), quant_scale(m));
    }
    if (t.lse && lane == 0) t.lse[int64_t(sp.row) * t.heads + h] = lse_of(top, sum);
  };
  if constexpr (WU == 1) {
    finish(ref, l, y);
  } else {
    float* mine = part + warp * (D + 2);
    if (lane == 0) mine[D] = ref, mine[D + 1] = l;
#pragma unroll
    for (int e = 0; e < E; e++) mine[d0 + e] = y[e];
    __syncthreads();
    if (warp != 0 && S == 1) return;
    float* block = part + WU * (D + 2);
    if (warp == 0) {
      float top = ninf(), sum = 0.f, val[E] = {};
      for (int w = 0; w < WU; w++) top = fmaxf(top, part[w * (D + 2) + D]);
      for (int w = 0; w < WU; w++) {
        const float* o1 = part + w * (D + 2);
        const float k = o1[D] == top ? 1.f : ex2(__fsub_rn(o1[D], top));
        sum = __fmaf_rn(k, o1[D + 1], sum);
#pragma unroll
        for (int e = 0; e < E; e++) val[e] = __fmaf_rn(k, o1[d0 + e], val[e]);
      }
      if (S == 1) {
        finish(top, sum, val);
        return;
      }
      if (lane == 0) block[D] = top, block[D + 1] = sum;
#pragma unroll
      for (int e = 0; e < E; e++) block[d0 + e] = val[e];
    }
    cluster_sync();
    if (rank == 0 && warp == 0) {
      float top = ninf(), sum = 0.f, val[E] = {};
      for (int n = 0; n < S; n++) top = fmaxf(top, peer_f32(block + D, n));
      for (int n = 0; n < S; n++) {
        const float m = peer_f32(block + D, n), k = m == top ? 1.f : ex2(__fsub_rn(m, top));
        sum = __fmaf_rn(k, peer_f32(block + D + 1, n), sum);
#pragma unroll
        for (int e = 0; e < E; e++) val[e] = __fmaf_rn(k, peer_f32(block + d0 + e, n), val[e]);
      }
      finish(top, sum, val);
    }
    cluster_sync();  // no block leaves while another reads its shared memory
  }
}

// Blocks and warps for a unit's keys: the stretches that they are cut into
// give the GPU enough warps, at most `longest` tiles of sixteen keys to one
// and at least two. With 64 tiles 48 ragged sequences of up to 12001 keys take
// 69 us, with 32 76, with 20 116: clusters grow that short sequences leave idle.
inline int64_t stretches(const Kv8Args& a, int64_t units, int warps_per_sm, int longest) {
  const int64_t tiles = (std::max(a.max_len, 1) + 15) / 16, most = std::max<int64_t>(1, tiles / 2);
  return std::min(most, std::max((tiles + longest - 1) / longest, (int64_t(kSMs) * warps_per_sm + units - 1) / units));
}
// Blocks of `warps` warps to a cluster that shares a unit's keys: as many as
// the parts ask for, of those that run at once (what
// cudaOccupancyMaxActiveClusters says on a B200, the only GPU that this is
// built for, of blocks of which an SM holds one or two). A second
// wave costs more than shorter stretches give: 4 sequences of 8192 tokens,
// 8 heads of 64 with 4 queries each, 36 us on clusters of 16 and 21 of 8.
inline int blocks_of(int64_t units, int64_t parts, int warps, int per_sm) {
  static constexpr int at_once[2][5] = {{148, 74, 33, 15, 7}, {296, 148, 71, 33, 14}};  // of 1, 2, 4, 8, 16
  int n = 0;
  while (n < 4 && (int64_t(warps) << n) < parts && units <= at_once[per_sm - 1][n + 1]) n++;
  return 1 << n;
}

template <int D, int NQ, int NP, int WU>
cudaError_t attend_launch(const Kv8Args& a, int type, const Kv8Attend& t, int64_t units, int qtiles, int S,
                          cudaStream_t st) {
  using Sh = Shape<D, NQ, WU>;
  const bool vec = type == 0 ? aligned<float>(t.q, 4) : aligned<__half>(t.q, 4);
  const bool ovec = type == 0 ? aligned<float>(t.out, 4) : aligned<__half>(t.out, 8);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(WU == 1 ? (units + Sh::warps - 1) / Sh::warps : units * S));
  cfg.blockDim = dim3(32 * Sh::warps);
  cfg.dynamicSmemBytes = Sh::smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(S);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_kv8_attend<D, NQ, NP, WU>, a, t, type, S, qtiles, int(units), vec, ovec);
}

// Warps of a block where a unit's keys are split over many.
template <int D>
constexpr int kWide = D == 64 ? 8 : 6;

template <int D, int NQ, int NP>
cudaError_t attend_t(const Kv8Args& a, int type, const Kv8Attend& t, cudaStream_t st) {
  const int group = t.heads / a.heads;
  const int qtiles = int((int64_t(a.max_new) * group + 8 * NQ - 1) / (8 * NQ));
  const int64_t units = int64_t(a.n) * a.heads * qtiles;
  const int64_t parts = stretches(a, units, 16, 64);
  if (parts == 1) return attend_launch<D, NQ, NP, 1>(a, type, t, units, qtiles, 1, st);
  // few units: wide blocks, two an SM; with more of them narrower ones are
  // the faster (48 sequences of 2000 keys and 4 heads: 40 us, wide ones 48)
  if constexpr (NQ == 1) {
    constexpr int WU = kWide<D>;
    if (parts > 4 && units <= kSMs)
      return attend_launch<D, NQ, NP, WU>(a, type, t, units, qtiles, blocks_of(units, parts, WU, 2), st);
  }
  // several queries: one wave again (16 sequences of 8192 keys, 4 heads, 16
  // queries: 53 us, with clusters of all the parts 101); one query a column,
  // whose blocks are smaller, gains from more (ragged: 69 us, one wave 123)
  int S = NQ > 1 ? blocks_of(units, parts, 4, 2) : 1;
  if (NQ == 1)
    while (S < 16 && S * 4 < parts) S *= 2;
  return attend_launch<D, NQ, NP, 4>(a, type, t, units, qtiles, S, st);
}

template <int D, int WU>
cudaError_t attend1_launch(const Kv8Args& a, int type, const Kv8Attend& t, int S, cudaStream_t st) {
  using Sh = Shape1<D, WU>;
  const int units = a.n * a.heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(WU == 1 ? (units + Sh::warps - 1) / Sh::warps : units * S));
  cfg.blockDim = dim3(32 * Sh::warps);
  cfg.dynamicSmemBytes = Sh::smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(S);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 1 : 0;
  const bool vec = type == 0 ? aligned<float>(t.q, 4) : aligned<__half>(t.q, 4);
  return cudaLaunchKernelEx(&cfg, k_kv8_attend1<D, WU>, a, t, type, S, units, vec);
}

template <int D>
cudaError_t attend1_d(const Kv8Args& a, int type, const Kv8Attend& t, cudaStream_t st) {
  const int64_t units = int64_t(a.n) * a.heads, parts = stretches(a, units, Shape1<D, 1>::per_sm, 64);
  if (parts == 1) return attend1_launch<D, 1>(a, type, t, 1, st);
  if (parts <= 4) return attend1_launch<D, 4>(a, type, t, 1, st);
  return attend1_launch<D, 8>(a, type, t, blocks_of(units, parts, 8, Shape1<D, 8>::blocks), st);
}

template <int D, int NP>
cudaError_t attend_d(const Kv8Args& a, int type, const Kv8Attend& t, cudaStream_t st) {
  const int64_t rows = int64_t(a.max_new) * (t.heads / a.heads);  // queries that share a head's keys
  if (rows == 1) return attend1_d<D>(a, type, t, st);
  if (rows <= 8) return attend_t<D, 1, NP>(a, type, t, st);
  // More than 32 queries go to the 5th-generation tensor core, 128 a block,
  // unless few blocks would have long stretches of keys that these kernels
  // split; more than 16 where one wave of blocks has few keys. 4 heads of 128,
  // bfloat16, us here and there: 64 queries of 16 sequences over 2048 keys 58
  // and 45, of 4 over 2048 31 and 45, over 512 26 and 23; 128 of 48 over 2048
  // 214 and 94; 32 of 16 over 512 29 and 24, over 2048 40 and 45, of 128 over
  // 512 67 and 72.
  const int64_t blocks = int64_t(a.n) * a.heads * ((rows + 127) / 128);
  const bool brief = a.max_len <= 512;
  if (rows > 32 ? brief || blocks >= kSMs / 4 : rows > 16 && brief && blocks <= kSMs)
    return launch_kv8_prompt(a, D, type, t, st);
  if (rows <= 16) return attend_t<D, 2, NP>(a, type, t, st);
  return attend_t<D, 4, NP>(a, type, t, st);
}

template <int D, int NQ, int NP, int WU>
void attend_attrs() {
  const auto k = k_kv8_attend<D, NQ, NP, WU>;
  cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape<D, NQ, WU>::smem));
  cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
template <int D, int WU>
void attend1_attrs() {
  cudaFuncSetAttribute(k_kv8_attend1<D, WU>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape1<D, WU>::smem));
  cudaFuncSetAttribute(k_kv8_attend1<D, WU>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
template <int D>
void attend1_init() {
  attend1_attrs<D, 1>();
  attend1_attrs<D, 4>();
  attend1_attrs<D, 8>();
}
template <int D, int NP>
void attend_init() {
  attend_attrs<D, 1, NP, 1>();
  attend_attrs<D, 1, NP, 4>();
  attend_attrs<D, 1, NP, kWide<D>>();
  attend_attrs<D, 2, NP, 1>();
  attend_attrs<D, 2, NP, 4>();
  attend_attrs<D, 4, NP, 1>();
  attend_attrs<D, 4, NP, 4>();
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8Args& a, int head_dim, int type, const Kv8Rows& k, const Kv8Rows& v,
                              cudaStream_t st) {
  if (head_dim == 64)
    return type == 0   ? append_t<64, float>(a, k, v, st)
           : type == 1 ? append_t<64, __half>(a, k, v, st)
                       : append_t<64, __nv_bfloat16>(a, k, v, st);
  return type == 0   ? append_t<128, float>(a, k, v, st)
         : type == 1 ? append_t<128, __half>(a, k, v, st)
                     : append_t<128, __nv_bfloat16>(a, k, v, st);
}

cudaError_t launch_kv8_read(const Kv8Args& a, int head_dim, int type, const Kv8Rows& k, const Kv8Rows& v,
                            cudaStream_t st) {
  if (head_dim == 64)
    return type == 0   ? read_t<64, float>(a, k, v, st)
           : type == 1 ? read_t<64, __half>(a, k, v, st)
                       : read_t<64, __nv_bfloat16>(a, k, v, st);
  return type == 0   ? read_t<128, float>(a, k, v, st)
         : type == 1 ? read_t<128, __half>(a, k, v, st)
                     : read_t<128, __nv_bfloat16>(a, k, v, st);
}

cudaError_t launch_kv8_attend(const Kv8Args& a, int head_dim, int type, const Kv8Attend& t, cudaStream_t st) {
  const cudaError_t e = head_dim == 64
                            ? (type == 0 ? attend_d<64, 2>(a, type, t, st) : attend_d<64, 1>(a, type, t, st))
                            : (type == 0 ? attend_d<128, 2>(a, type, t, st) : attend_d<128, 1>(a, type, t, st));
  if (e != cudaSuccess) cudaGetLastError();  // returned: a later launch must not find it as its own
  return e;
}

cudaError_t launch_kv8_copy_pages(const Kv8Args& a, int head_dim, int layers, const int* from, const int* to, int count,
                                  cudaStream_t st) {
  k_kv8_copy_pages<<<dim3(count, layers), 256, 0, st>>>(a, (a.heads << a.plog) * head_dim, from, to);
  return cudaGetLastError();
}

void kv8_kernels_init() {
  kv8_prompt_init();
  attend1_init<64>();
  attend1_init<128>();
  attend_init<64, 2>();
  attend_init<64, 1>();
  attend_init<128, 2>();
  attend_init<128, 1>();
}

}  // namespace grx
