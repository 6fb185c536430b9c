// Attention over the 8-bit paged cache for prompts: many queries of a
// sequence share a key head, so the products belong on the 5th-generation
// tensor core (tcgen05.mma, accumulators in Tensor Memory).
//
// A block takes 128 query rows (token by token, the heads of a group side by
// side) against tiles of 64 keys, one pass with the running maximum and sum:
//  * warps 8-15 turn a tile's bytes into float16 operands (exact): the keys
//    as they lie, [key][value], the values turned, [value][key], both in the
//    128-byte swizzle that the tensor core reads; the next tile's bytes come
//    into registers meanwhile;
//  * warp 16 issues the products: scores S = Q·Kᵀ into one of two TMEM tiles,
//    Q being the sum of two float16s of a row scaled to 2^14 (22 bits and
//    more: 32-bit scores), and O += P·V with P from TMEM, one float16 for
//    16-bit outputs and the sum of two for float32 ones. The scores of tile
//    j + 2 are issued ahead of the outputs of tile j;
//  * warps 0-3 take the even tiles and warps 4-7 the odd ones, a thread to a
//    row and with a maximum, a sum and an O of their own, joined at the end:
//    the scores' maximum from TMEM, the scores again, weights 2^11·p·s_v/W,
//    written back as P, W being the row's own, at least a sixteenth of its
//    largest p·s_v so far: a weight is off by 2^-12 of itself (2^-22 as the
//    sum of two), or by 2^-36 W where that is more. The maximum moves only when a
//    score passes it by 2^8; when a weight passes W by 2^4, the row of O in
//    TMEM is multiplied. So one half's exponentials run while the other half
//    waits.
// Blocks with the most keys start first. Every wait is bounded (about a
// second of clocks); one that runs out sets the block's `dead` word, every
// role leaves its loop, the block frees its TMEM, and the status word gets
// GRX_ETIMEDOUT.
//
// Heads of 128, bfloat16: 1.06 us for a tile of a block and 9 us for a block's
// beginning and end; 8 prompts of 1 to 512 tokens with 300 to 2500 keys,
// 4 heads with 4 queries each: 88 us, 0.32 PFLOP/s counted as float16 products
// once. Of a tile's 2000 clocks the products take 1200 (Q's two halves from
// shared memory, 128 bytes a clock), the conversions and exponentials run
// beside them; what is left is the roles' waits for one another.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "kv8.cuh"

namespace grx {

namespace {

constexpr int kTimedOut = -7;  // GRX_ETIMEDOUT
constexpr int kRows = 128, kKeys = 64;
constexpr float kTo14 = 1.f / 256.f;  // from kQueryUnits to 2^14

__device__ __forceinline__ uint32_t smem_at(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded; false once about 2^31 clocks have passed or another role gave up.
// All lanes of a warp get the same answer.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  bool ok = bar_try(bar, parity);
  if (!ok) {
    const long long t0 = clock64();
    while (!(ok = bar_try(bar, parity))) {
      if (*dead) break;
      if (clock64() - t0 > (1LL << 31)) {
        *dead = 1;
        break;
      }
    }
  }
  return __all_sync(FULL, ok);
}
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// Executed by a whole warp in step, issued by the one lane elect.sync picks.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n"
      "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar)
      : "memory");
}
// K-major operand in the 128-byte swizzle: rows of 128 bytes, groups of 8
// rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// D (+)= A·Bᵀ, float16 operands, float32 sums; A in shared memory or TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(int(add))
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(int(add))
      : "memory");
}
// 32 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* d) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]), "=r"(d[8]),
        "=r"(d[9]), "=r"(d[10]), "=r"(d[11]), "=r"(d[12]), "=r"(d[13]), "=r"(d[14]), "=r"(d[15]), "=r"(d[16]),
        "=r"(d[17]), "=r"(d[18]), "=r"(d[19]), "=r"(d[20]), "=r"(d[21]), "=r"(d[22]), "=r"(d[23]), "=r"(d[24]),
        "=r"(d[25]), "=r"(d[26]), "=r"(d[27]), "=r"(d[28]), "=r"(d[29]), "=r"(d[30]), "=r"(d[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* d) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(at),
      "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]), "r"(d[4]), "r"(d[5]), "r"(d[6]), "r"(d[7]), "r"(d[8]), "r"(d[9]),
      "r"(d[10]), "r"(d[11]), "r"(d[12]), "r"(d[13]), "r"(d[14]), "r"(d[15]), "r"(d[16]), "r"(d[17]), "r"(d[18]),
      "r"(d[19]), "r"(d[20]), "r"(d[21]), "r"(d[22]), "r"(d[23]), "r"(d[24]), "r"(d[25]), "r"(d[26]), "r"(d[27]),
      "r"(d[28]), "r"(d[29]), "r"(d[30]), "r"(d[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* d) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(at),
      "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]), "r"(d[4]), "r"(d[5]), "r"(d[6]), "r"(d[7]), "r"(d[8]), "r"(d[9]),
      "r"(d[10]), "r"(d[11]), "r"(d[12]), "r"(d[13]), "r"(d[14]), "r"(d[15])
      : "memory");
}
__device__ __forceinline__ uint32_t to_f16(uint32_t u) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(u ^ 0x64806480u), "r"(0xe480e480u));
  return d;
}
__device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// NP: float16s of a weight.
template <int D, int NP>
struct Prompt {
  static constexpr int threads = 544;
  // shared memory: bytes of the two halves of Q, of a tile's keys and values
  static constexpr int q = kRows * D * 2, k = kKeys * D * 2, v = D * kKeys * 2;
  static constexpr int stages = 4;  // tiles of operands
  static constexpr int off_k = 2 * q, off_v = off_k + stages * k, off_s = off_v + stages * v;  // scales: [4][4] pairs
  static constexpr int off_f = off_s + 4 * 4 * 8, off_x = off_f + kRows * 4;  // rows' factors; the halves' {maximum, sum, W}
  static constexpr int off_bar = off_x + 2 * 3 * kRows * 4, used = off_bar + 14 * 8 + 16;
  // TMEM columns: two score tiles, two weight tiles, two halves' outputs: all
  // there are, or more than half of them
  static constexpr int c_p = 2 * kKeys, c_o = c_p + 2 * NP * kKeys / 2, columns = 512;
  static_assert(c_o + 2 * D <= columns);
  // so an SM holds one block: more than half of its shared memory
  static constexpr int half_sm = 115 * 1024;
  static constexpr int smem = 1024 + (used > half_sm ? used : half_sm);
};

template <int D, int NP>
__global__ void __launch_bounds__(544, 1)
    k_kv8_prompt(Kv8Args a, Kv8Attend t, int type, int qtiles, bool vec, bool ovec) {
  using C = Prompt<D, NP>;
  constexpr int H2 = D / 64;
  extern __shared__ uint8_t raw_smem[];
  const uint32_t raw = smem_at(raw_smem), base = (raw + 1023) & ~1023u;
  uint8_t* mem = raw_smem + (base - raw);
  float2* scales = reinterpret_cast<float2*>(mem + C::off_s);  // [tile & 3][sixteen keys]
  float* rowf = reinterpret_cast<float*>(mem + C::off_f);
  float* halves = reinterpret_cast<float*>(mem + C::off_x);  // [half][3][row]
  const uint32_t bars = base + C::off_bar;
  // Barriers of tile j, and the parity that they end with: its operands and
  // scales are in shared memory; its scores in S j & 1; its weights in P j & 1;
  // its outputs in O j & 1. No role is four tiles ahead of another.
  const auto conv = [&](int j) { return bars + 8 * (j & 3); };
  const auto added = [&](int j) { return bars + 8 * (4 + (j & 3)); };
  const auto scored = [&](int j) { return bars + 8 * (8 + (j & 1)); };
  const auto weighed = [&](int j) { return bars + 8 * (10 + (j & 1)); };
  const auto taken = [&](int j) { return bars + 8 * (12 + (j & 1)); };  // scores read for the last time
  const auto of4 = [](int j) { return uint32_t(j >> 2) & 1u; };
  const auto of2 = [](int j) { return uint32_t(j >> 1) & 1u; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mem + C::off_bar + 112);
  volatile int* dead = reinterpret_cast<volatile int*>(mem + C::off_bar + 116);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // heads of one tile side by side, the last queries (the most keys) first
  const int h = blockIdx.x % a.heads, rest = blockIdx.x / a.heads, i = rest % a.n, qt = qtiles - 1 - rest / a.n;
  const int group = t.heads / a.heads;
  const Kv8Span sp = kv8_span(a, i);
  if (!sp.ok) {
    if (tid == 0) report(a);
    return;
  }
  const int r0 = qt * kRows, nrow = min(kRows, sp.T * group - r0);
  if (nrow <= 0) return;
  const int p0 = sp.len - sp.T;
  const int pmin = p0 + r0 / group, pmax = p0 + (r0 + nrow - 1) / group;
  const int first = a.first ? max(0, a.first[i]) : 0;
  const int klo = max(first, t.window > 0 ? pmin - t.window + 1 : 0);
  const int tb = klo / kKeys, nt = max(0, (pmax + kKeys) / kKeys - tb);  // tiles tb .. tb + nt − 1

  if (tid == 0) {
    *dead = 0;
    for (int j = 0; j < 4; j++) {
      bar_init(conv(j), 8);
      bar_init(added(j), 1);
    }
    for (int j = 0; j < 2; j++) {
      bar_init(scored(j), 1);
      bar_init(weighed(j), 4);
      bar_init(taken(j), 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 16) {
    asm volatile(
        "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
        "tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::"r"(smem_at(tmem_slot)),
        "r"(C::columns)
        : "memory");
  }

  // --- the queries: rotated, scaled, as the sum of two float16s; four lanes
  // to a row, eight rows to a warp ---
  const auto queries = [&]() {
    const int g = lane >> 2, tg = lane & 3;
    {
      const int r = warp * 8 + g;
      const bool there = r < nrow;
      const int tq = there ? (r0 + r) / group : 0, hq = h * group + (there ? (r0 + r) % group : 0);
      float x[H2][16];
      const int64_t off = int64_t(sp.row + tq) * t.q.row + int64_t(hq) * t.q.head + 16 * tg;
      load_row<D>(t.q.p, off, type, vec, there, x);
      rotate16<D>(x, a, p0 + tq, tg);
      const float amax = group_amax<D>(x, FULL);
      // the sign of the scale goes into the query, so that the row's factor has none
      const float to = __fmul_rn(lift_row<D>(x, amax), t.scale < 0.f ? -kTo14 : kTo14);
#pragma unroll
      for (int j = 0; j < H2; j++) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          // a row that is no number: 0 here, and its factor is none
          const float y0 = to != 0.f ? __fmul_rn(x[j][2 * e], to) : 0.f, y1 = to != 0.f ? __fmul_rn(x[j][2 * e + 1], to) : 0.f;
          hi[e] = pack_f16(y0, y1);
          lo[e] = pack_f16(__fsub_rn(y0, __half2float(__ushort_as_half(hi[e] & 0xffff))),
                           __fsub_rn(y1, __half2float(__ushort_as_half(hi[e] >> 16))));
        }
        const uint32_t at = base + j * (kRows * 128) + r * 128;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const uint32_t o = at + ((2 * tg + c) ^ (r & 7)) * 16;
          sts16(o, hi[4 * c], hi[4 * c + 1], hi[4 * c + 2], hi[4 * c + 3]);
          sts16(o + C::q, lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
        }
      }
      if (tg == 0)
        rowf[r] = __fmul_rn(__fmul_rn(amax, 256.f / kQueryUnits), __fmul_rn(fabsf(t.scale), 1.44269504f));
    }
    fence_async();
  };
  // the set-up is done: barriers, TMEM, queries
  uint32_t tmem = 0;
  const auto ready = [&]() {
    fence_before();
    __syncthreads();
    fence_after();
    tmem = *tmem_slot;
  };

  if (warp == 16) {
    ready();
    // ---- the products
    const uint32_t idesc_s = (1u << 4) | (uint32_t(kKeys >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
    const uint32_t idesc_o = (1u << 4) | (uint32_t(D >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
    const auto outputs = [&](int j) {
      const int b = j & 1;
      fence_after();
#pragma unroll
      for (int n = 0; n < NP; n++)
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; kk++)
          mma_ts(tmem + C::c_o + b * D, tmem + C::c_p + (b * NP + n) * (kKeys / 2) + kk * 8,
                 operand(base + C::off_v + j % C::stages * C::v + kk * 32), idesc_o, j > 1 || n > 0 || kk > 0);
      commit(added(j));
    };
    int done = 0;
    bool ok = true;
    for (int j = 0; j < nt && ok; j++) {
      const int b = j & 1;
      ok = bar_wait(conv(j), of4(j), dead) && (j < 2 || bar_wait(taken(j - 2), of2(j - 2), dead));
      if (!ok) break;
      fence_after();
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int kk = 0; kk < D / 16; kk++)
          mma_ss(tmem + b * kKeys, operand(base + n * C::q + (kk / 4) * (kRows * 128) + (kk % 4) * 32),
                 operand(base + C::off_k + j % C::stages * C::k + (kk / 4) * (kKeys * 128) + (kk % 4) * 32),
                 idesc_s,
                 n > 0 || kk > 0);
      commit(scored(j));
      if (j > 1) {
        ok = bar_wait(weighed(j - 2), of2(j - 2), dead);
        if (ok) outputs(j - 2), done = j - 1;
      }
    }
    for (int j = max(nt - 2, 0); j < nt && ok; j++) {
      ok = bar_wait(weighed(j), of2(j), dead);
      if (ok) outputs(j), done = j + 1;
    }
    if (done < nt && nt > 0) {
      // given up: what was issued ends before the TMEM is released
      commit(added(0));
      const long long t0 = clock64();
      while (clock64() - t0 < (1LL << 24)) {
      }
    }
  } else if (warp >= 8) {
    // ---- a tile's operands
    const int ct = tid - 256;  // 0 .. 255
    constexpr int KU = D / 64;  // sixteen-byte units of keys a thread
    const bool turns = D == 128 || ct < 128;  // has a unit of eight tokens by four values
    const int64_t pbytes = int64_t(a.heads << a.plog) * D;
    const int8_t* kh = a.k + (int64_t(h) << a.plog) * D;
    const int8_t* vh = a.v + (int64_t(h) << a.plog) * D;
    // lane l holds page and scales of the sixteen keys 16·(base + l) .., eight
    // tiles at a time, and the pages of the next eight
    const int plast = (sp.len + 15) >> 4;
    const auto page_of = [&](int c) { return c < plast ? kv8_page(a, i, c >> (a.plog - 4)) : -1; };
    // −inf where there is no page
    const auto scale_of = [&](int page) {
      if (page < 0) return make_float2(ninf(), 0.f);
      return sound_scales(reinterpret_cast<const float2*>(a.scale)[int64_t(page) * a.heads + h]);
    };
    int c0 = tb * 4, page = page_of(c0 + lane), ahead = page_of(c0 + 32 + lane);
    if (page < 0 && c0 + lane < plast && c0 + lane <= pmax >> 4) report(a);
    float2 scale = scale_of(page), scale_ahead = scale;
    struct Bytes {
      uint4 k[KU];
      uint32_t v[8];
      float2 scale;
    } one, two;  // two tiles' bytes are under way: a tile takes less than a load's way to memory
    const auto load = [&](int j, Bytes& to) {
      int64_t at16[4];  // where the tile's four groups of sixteen keys lie (some page's bytes where there is none)
      const int c = (tb + j) * 4;
      if (c - c0 == 32) {
        c0 += 32;
        page = ahead;
        if (page < 0 && c0 + lane < plast && c0 + lane <= pmax >> 4) report(a);
        scale = scale_ahead;
        ahead = page_of(c0 + 32 + lane);
      }
      if (c - c0 == 16) scale_ahead = scale_of(ahead);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int pg = __shfl_sync(FULL, page, c - c0 + u);
        at16[u] = int64_t(max(pg, 0)) * pbytes + ((c + u) * 16 & ((1 << a.plog) - 1)) * D;
      }
      to.scale.x = __shfl_sync(FULL, scale.x, c - c0 + (lane & 3));
      to.scale.y = __shfl_sync(FULL, scale.y, c - c0 + (lane & 3));
#pragma unroll
      for (int u = 0; u < KU; u++) {
        const int n = ct + 256 * u, key = n / (D / 16), g16 = key >> 4;  // unit: key, sixteen values n % (D/16)
        const int64_t at = D == 128 ? (g16 & 1 ? at16[2 * u + 1] : at16[2 * u])
                                    : (g16 & 2 ? (g16 & 1 ? at16[3] : at16[2]) : (g16 & 1 ? at16[1] : at16[0]));
        to.k[u] = __ldg(reinterpret_cast<const uint4*>(kh + at + (key & 15) * D + n % (D / 16) * 16));
      }
      if (turns) {
        const int grp = ct / (D / 4), g16 = grp >> 1;  // unit: tokens 8·grp .., values 4·(ct % (D/4)) ..
        const int64_t at = g16 & 2 ? (g16 & 1 ? at16[3] : at16[2]) : (g16 & 1 ? at16[1] : at16[0]);
        const int8_t* from = vh + at + (grp & 1) * 8 * D + ct % (D / 4) * 4;
#pragma unroll
        for (int e = 0; e < 8; e++) to.v[e] = __ldg(reinterpret_cast<const uint32_t*>(from + e * D));
      }
    };
    const auto turn = [&](int j, Bytes& in) {
      if (j >= C::stages && !bar_wait(added(j - C::stages), of4(j - C::stages), dead)) return false;
      const uint32_t kst = base + C::off_k + j % C::stages * C::k, vst = base + C::off_v + j % C::stages * C::v;
      if (ct < 4) scales[(j & 3) * 4 + ct] = in.scale;
#pragma unroll
      for (int u = 0; u < KU; u++) {
        const int n = ct + 256 * u, key = n / (D / 16), c = n % (D / 16);  // values 16c .. : chunks 2c and 2c + 1
        const uint32_t at = kst + (c / 4) * (kKeys * 128) + key * 128;
        const int swap = D == 128 ? c >> 2 & 1 : key & 1;  // neighbours write different banks
        const uint32_t w[4] = {in.k[u].x, in.k[u].y, in.k[u].z, in.k[u].w};
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int s = e ^ swap;
          const uint32_t x = s ? w[2] : w[0], y = s ? w[3] : w[1];
          sts16(at + ((2 * (c % 4) + s) ^ (key & 7)) * 16, to_f16(__byte_perm(x, 0, 0x4140)),
                to_f16(__byte_perm(x, 0, 0x4342)), to_f16(__byte_perm(y, 0, 0x4140)), to_f16(__byte_perm(y, 0, 0x4342)));
        }
      }
      if (turns) {
        const int grp = ct / (D / 4), w = ct % (D / 4);
        const uint32_t at = vst + 4 * w * 128;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int v = (e + (w >> 1)) & 3;  // the order in which neighbours write different banks
          const uint32_t pick = v | (4 + v) << 8;
          uint32_t y[4];
#pragma unroll
          for (int m = 0; m < 4; m++) y[m] = to_f16(__byte_perm(in.v[2 * m], in.v[2 * m + 1], pick) & 0x00ff00ffu);
          sts16(at + v * 128 + (grp ^ ((4 * w + v) & 7)) * 16, y[0], y[1], y[2], y[3]);
        }
      }
      fence_async();
      __syncwarp();
      if (lane == 0) bar_arrive(conv(j));
      if (j + 2 < nt) load(j + 2, in);
      return true;
    };
    if (nt > 0) load(0, one);
    if (nt > 1) load(1, two);
    queries();
    ready();
    for (int j = 0; j < nt; j += 2)
      if (!turn(j, one) || (j + 1 < nt && !turn(j + 1, two))) break;
  } else {
    // ---- the rows: a half of the tiles each
    queries();
    ready();
    const int quarter = warp & 3, half = warp >> 2, r = quarter * 32 + lane;
    const bool there = r < nrow;
    const int tq = there ? (r0 + r) / group : 0, hq = h * group + (there ? (r0 + r) % group : 0);
    const int p = there ? p0 + tq : pmax;
    const int lo = max(first, t.window > 0 ? p - t.window + 1 : 0);  // sees lo .. p
    const int in_lo = max(first, t.window > 0 ? pmax - t.window + 1 : 0);
    const float f = rowf[r];
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t my_s = lanes + half * kKeys, my_o = lanes + C::c_o + half * D;
    const uint32_t my_p = lanes + C::c_p + half * NP * (kKeys / 2);
    float ref = ninf(), l = 0.f, toW = pow2(253), most = ninf();  // 2^11/W, log2 of 2^4·W
    bool ok = true;
    for (int j = half; j < nt; j += 2) {
      const int key0 = (tb + j) * kKeys;
      ok = bar_wait(conv(j), of4(j), dead) && bar_wait(scored(j), of2(j), dead);
      if (!ok) break;
      fence_after();
      float2 c[4];
      uint32_t turned = 0;  // groups of sixteen keys whose scale is below 0: their products change sign, the scale has none
#pragma unroll
      for (int g = 0; g < 4; g++) {
        c[g] = scales[(j & 3) * 4 + g];
        if (c[g].x < 0.f && c[g].x != ninf()) {
          turned |= 1u << g;
          c[g].x = -c[g].x;
        }
      }
      // the 32 products of half u of the tile
      const auto turn = [&](int u, float* x) {
#pragma unroll
        for (int g = 0; g < 2; g++)
          if (turned >> (2 * u + g) & 1) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[16 * g + e] = -x[16 * g + e];
          }
      };
      const bool edge = c[0].x == ninf() || c[1].x == ninf() || c[2].x == ninf() || c[3].x == ninf() || key0 < in_lo ||
                        key0 + kKeys - 1 > pmin;
      // bit e: this row sees key e of the tile
      uint64_t seen = ~0ull;
      if (edge) {
        const int from = max(lo - key0, 0), to = min(p - key0, kKeys - 1);
        seen = from > to ? 0 : (~0ull >> (kKeys - 1 - to)) >> from << from;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          if (c[g].x == ninf()) seen &= ~(0xffffull << (16 * g));
        }
      }
      const auto hidden = [&](int e) { return !(uint32_t(e < 32 ? seen : seen >> 32) >> (e & 31) & 1); };
      uint32_t s[32];
      f2* x2 = reinterpret_cast<f2*>(s);
      float* x = reinterpret_cast<float*>(s);
      // the largest score: a group's largest product times its factor, from
      // which every sign has been taken
      float top = ninf(), heavy = ninf();  // and the largest of log2 of a weight, from the same
#pragma unroll
      for (int u = 0; u < 2; u++) {
        tmem_ld32(my_s + 32 * u, s);
        wait_ld();
        if (turned) turn(u, x);
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (hidden(32 * u + e)) x[e] = ninf();
        }
#pragma unroll
        for (int g = 0; g < 2; g++) {
          float m[4];
#pragma unroll
          for (int e = 0; e < 4; e++)
            m[e] = fmaxf(fmaxf(x[16 * g + e], x[16 * g + 4 + e]), fmaxf(x[16 * g + 8 + e], x[16 * g + 12 + e]));
          float y = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
          if (y != ninf()) y = __fmul_rn(y, __fmul_rn(f, c[2 * u + g].x));
          top = fmaxf(top, y);
          heavy = fmaxf(heavy, __fadd_rn(y, lg2(c[2 * u + g].y)));
        }
      }
      if (j > 1) {
        ok = bar_wait(added(j - 2), of4(j - 2), dead);  // P is free, O as it was left
        if (!ok) break;
        fence_after();
      }
      // the references move: a score 2^8 above the row's (any, before its
      // first key), a weight 2^4 above W
      const bool over = top > __fadd_rn(ref, 8.f);
      if (__any_sync(FULL, over || __fsub_rn(heavy, ref) > most)) {
        float unit = inverse<NP>(toW);  // O's, 2^-11 W
        if (over) {
          const float up = ex2(__fsub_rn(ref, top));
          ref = top;
          l = __fmul_rn(l, up);
          unit = __fmul_rn(unit, up);  // what it is worth now
        }
        toW = weight_scale<NP>(fmaxf(__fmul_rn(unit, 2048.f), ex2(__fsub_rn(heavy, ref))), &most);
        const float k = __fmul_rn(unit, toW);
        if (j > 1) {
#pragma unroll 1
          for (int n = 0; n < D; n += 32) {
            tmem_ld32(my_o + n, s);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; e++) x[e] = __fmul_rn(x[e], k);
            tmem_st32(my_o + n, s);
          }
          wait_st();
        }
      }
      const f2 m = f2dup(ref == ninf() ? 0.f : -ref);
      f2 sum = 0;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        tmem_ld32(my_s + 32 * u, s);
        wait_ld();
        if (u == 1) {  // the tile after next may come into their place
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(taken(j));
        }
        if (turned) turn(u, x);
        const float2 c0 = c[2 * u], c1 = c[2 * u + 1];
        const f2 f0 = f2dup(__fmul_rn(f, c0.x)), f1 = f2dup(__fmul_rn(f, c1.x));
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const f2 y = f2fma(x2[e], e < 8 ? f0 : f1, m);
          x2[e] = f2make(ex2(f2lo(y)), ex2(f2hi(y)));
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 32; e++)
            if (hidden(32 * u + e)) x[e] = 0.f;
        }
        // (a scale far above W has terms of 0, or as far below 1: no infinity here)
        const f2 w0 = f2dup(fminf(__fmul_rn(c0.y, toW), 3.4e38f)), w1 = f2dup(fminf(__fmul_rn(c1.y, toW), 3.4e38f));
#pragma unroll
        for (int e = 0; e < 16; e++) {
          sum = f2add(sum, x2[e]);
          x2[e] = f2mul(x2[e], e < 8 ? w0 : w1);
        }
#pragma unroll
        for (int n = 0; n < NP; n++) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; e++) {
            w[e] = pack_f16(x[2 * e], x[2 * e + 1]);
            if (n + 1 < NP) {
              x[2 * e] = __fsub_rn(x[2 * e], __half2float(__ushort_as_half(w[e] & 0xffff)));
              x[2 * e + 1] = __fsub_rn(x[2 * e + 1], __half2float(__ushort_as_half(w[e] >> 16)));
            }
          }
          tmem_st16(my_p + n * (kKeys / 2) + 16 * u, w);
        }
      }
      l = __fadd_rn(l, __fadd_rn(f2lo(sum), f2hi(sum)));
      wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(weighed(j));
    }
    // the halves together; a half without a tile has no O
    if (ok && nt > 0) ok = bar_wait(added(nt - 1), of4(nt - 1), dead);
    if (ok && nt > 1) ok = bar_wait(added(nt - 2), of4(nt - 2), dead);
    halves[(half * 3 + 0) * kRows + r] = ref;
    halves[(half * 3 + 1) * kRows + r] = l;
    halves[(half * 3 + 2) * kRows + r] = inverse<NP>(toW);
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    if (ok) {
      fence_after();
      const float ref0 = halves[r], ref1 = halves[3 * kRows + r], l0 = halves[kRows + r], l1 = halves[4 * kRows + r];
      ref = fmaxf(ref0, ref1);
      const float k0 = ref0 == ref ? 1.f : ex2(__fsub_rn(ref0, ref)), k1 = ref1 == ref ? 1.f : ex2(__fsub_rn(ref1, ref));
      l = __fadd_rn(__fmul_rn(l0, k0), __fmul_rn(l1, k1));
      // a row without keys has an O of zeros or none
      const float inv0 = l == 0.f ? 0.f : __fdiv_rn(__fmul_rn(halves[2 * kRows + r], k0), l);
      const float inv1 = l == 0.f ? 0.f : __fdiv_rn(__fmul_rn(halves[5 * kRows + r], k1), l);
#pragma unroll 1
      for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
        uint32_t o[32] = {}, o1[32] = {};
        if (nt > 0) tmem_ld32(lanes + C::c_o + c, o);
        if (nt > 1) tmem_ld32(lanes + C::c_o + D + c, o1);
        wait_ld();
        float* y = reinterpret_cast<float*>(o);
#pragma unroll
        for (int e = 0; e < 32; e++) y[e] = __fadd_rn(__fmul_rn(y[e], inv0), __fmul_rn(__uint_as_float(o1[e]), inv1));
        // into the place of Q, chunks of 16 bytes in an order that keeps banks apart
#pragma unroll
        for (int e = 0; e < 8; e++)
          sts16(base + r * (D * 4) + ((c / 4 + e) ^ (r & 7)) * 16, o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        if (t.q8 && there) {  // one Q8_0 block
          const int64_t to = (int64_t(sp.row + tq) * t.heads + hq) * D + c;
          float most = 0.f;
          uint32_t w[8] = {};
#pragma unroll
          for (int e = 0; e < 32; e++) most = fmaxf(most, fabsf(y[e]));
#pragma unroll
          for (int e = 0; e < 32; e++) w[e / 4] |= uint32_t(uint8_t(quant_val(y[e], most))) << (8 * (e % 4));
          uint4* op = reinterpret_cast<uint4*>(t.q8 + to);
          op[0] = make_uint4(w[0], w[1], w[2], w[3]);
          op[1] = make_uint4(w[4], w[5], w[6], w[7]);
          t.q8s[to / QK] = make_float2(quant_scale(most), quant_scale(most));
        }
      }
      if (there && half == 0 && t.lse) t.lse[int64_t(sp.row + tq) * t.heads + hq] = lse_of(ref, l);
    }
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    if (ok && t.out.p) {
      // whole rows to memory, sixteen to a warp
      constexpr int E = NP == 2 ? 4 : 8, L = D / E;  // values a lane, lanes a row
      const float* stage = reinterpret_cast<const float*>(mem);
      const int own = warp * 16 + (lane & 15), n = min(r0 + own, r0 + nrow - 1);
      const int64_t to = int64_t(sp.row + n / group) * t.out.row + int64_t(h * group + n % group) * t.out.head;
#pragma unroll 4
      for (int i16 = 0; i16 < 16; i16 += 32 / L) {
        const int row = warp * 16 + i16 + lane / L, c = lane % L * E;
        const int64_t at = __shfl_sync(FULL, to, i16 + lane / L) + c;
        if (row >= nrow) continue;
        float y[E];
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(y + e) =
              *reinterpret_cast<const float4*>(stage + row * D + ((c + e) / 4 ^ (row & 7)) * 4);
        if (!ovec) {
#pragma unroll
          for (int e = 0; e < E; e++) put(t, type, at + e, y[e]);
        } else if (NP == 2) {
          *reinterpret_cast<float4*>(static_cast<float*>(const_cast<void*>(t.out.p)) + at) = *reinterpret_cast<float4*>(y);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; e++)
            w[e] = type == 1 ? pack_f16(y[2 * e % E], y[(2 * e + 1) % E])
                             : uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(y[2 * e % E]))) |
                                   uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(y[(2 * e + 1) % E]))) << 16;
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(const_cast<void*>(t.out.p)) + at) =
              make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 16) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(C::columns) : "memory");
  }
  if (tid == 0 && *dead && a.status) *a.status = kTimedOut;
}

template <int D, int NP>
cudaError_t launch_t(const Kv8Args& a, int type, const Kv8Attend& t, cudaStream_t st) {
  using C = Prompt<D, NP>;
  const int qtiles = int((int64_t(a.max_new) * (t.heads / a.heads) + kRows - 1) / kRows);
  const bool vec = type == 0 ? aligned<float>(t.q, 4) : aligned<__half>(t.q, 4);
  const bool ovec = type == 0 ? aligned<float>(t.out, 4) : aligned<__half>(t.out, 8);
  k_kv8_prompt<D, NP><<<unsigned(int64_t(qtiles) * a.n * a.heads), C::threads, C::smem, st>>>(a, t, type, qtiles, vec, ovec);
  return cudaGetLastError();
}

template <int D, int NP>
void init_t() {
  cudaFuncSetAttribute(k_kv8_prompt<D, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Prompt<D, NP>::smem);
}

}  // namespace

cudaError_t launch_kv8_prompt(const Kv8Args& a, int head_dim, int type, const Kv8Attend& t, cudaStream_t st) {
  if (head_dim == 64) return type == 0 ? launch_t<64, 2>(a, type, t, st) : launch_t<64, 1>(a, type, t, st);
  return type == 0 ? launch_t<128, 2>(a, type, t, st) : launch_t<128, 1>(a, type, t, st);
}

void kv8_prompt_init() {
  init_t<64, 1>();
  init_t<64, 2>();
  init_t<128, 1>();
  init_t<128, 2>();
}

}  // namespace grx
