// Beam search: selection over beams and vocabulary, reordering of per-beam state in place,
// and the back-trace of the written sequences (include/xgraph_b200.h has the definitions).
#include "beams.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <atomic>
#include <cfloat>
#include <string>

extern "C" int xg_set_error(int code, const char* message);

namespace xg {
namespace beams {
namespace {

constexpr uint32_t kFull = 0xffffffffu;

// ---------------------------------------------------------------------------------------
// Selection, first kernel: every row's log-sum parts and its best tokens.
//
// A CTA streams a share of one row in steps of kVecs 16-byte vectors a thread.  The vectors go
// through a ring in shared memory that each thread fills (cp.async, two steps ahead) and reads
// for itself, so loads stay in flight while a step is computed on and no register holds them.
// Each logit is read once: a step adds its exponentials to the thread's sum and leaves the
// maximum of the thread's vectors in shared memory.  The best tokens lie in the few entries of
// that table whose maximum is among its best; those alone are read again for their tokens.
// (Listing candidate vectors against a running bound instead cost a barrier a step and, in most
// warp-steps, a divergent push: 31 us against 25 for 256 rows of 128,256 bf16.)
//
// What bounds it: a CTA's fixed way -- flags, mask words, first data, then the bound, the entries
// and their tokens, some 7 us of latencies -- around its stream, which runs at the SM's share of
// the memory rate.  256 rows of 128,256 bf16 (a fifth of them ended, 52 MB): both kernels 23.2 us
// where the bytes take 8.0; the stream is 8 of them, the exponentials' unit 3, the launches and
// the merge 6.  Masked rows are also bound by instructions where a mask is mixed (the bits' spread
// and the blend): 27.5 us, 5.8 for the bytes.

constexpr int32_t kScanThreads = 256;
constexpr int32_t kScanWarps = kScanThreads / 32;
constexpr int32_t kVecs = 4;          // 16-byte vectors of a thread in one step: an entry of the table
constexpr int32_t kSteps = 2;         // steps in the ring
constexpr int32_t kRound = 16;        // steps of the table; after as many the best tokens are taken out
constexpr int32_t kListCap = 512;     // entries read again; see list_crowded for why they suffice
constexpr int32_t kPushCap = 1024;    // tokens (keys) of the listed entries
constexpr int32_t kRankMost = kScanThreads;  // keys put in order by counting
constexpr float kFar = 65536.0f;      // logits of this magnitude take the difference from the maximum first
constexpr int32_t kPoolMax = 8192;    // candidates of a group that the second kernel takes

// Floats as unsigned integers of the same order (-0 made +0 by the caller).
__device__ __forceinline__ uint32_t rising(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_rising(uint32_t o) {
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : kFull));
}
constexpr uint32_t kRisingLowest = 0x00800000u;  // rising(-FLT_MAX); -inf lies below it

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {  // within 2^-22 of 2^x, relatively
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  return static_cast<uint64_t>(__float_as_uint(a)) | (static_cast<uint64_t>(__float_as_uint(b)) << 32);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float low(uint64_t a) { return __uint_as_float(static_cast<uint32_t>(a)); }
__device__ __forceinline__ float high(uint64_t a) { return __uint_as_float(static_cast<uint32_t>(a >> 32)); }

constexpr float kLog2eHi = 1.44269502162933349609375f;  // log2(e) in two floats
constexpr float kLog2eLo = 1.92596299112661746887e-8f;
// An anchor's natural logarithm: sums are of 2^(x kLog2eHi - anchor), so of exp(x - ref), nearly,
// with the ref at which x kLog2eHi is the anchor.
constexpr double kAnchorLn = 1.0 / static_cast<double>(kLog2eHi);
constexpr float kAbove = 8.0f;  // a warp's maximum stands up to this much above its anchor

// How the three logit types sit in a 16-byte vector.
struct F32 {
  static constexpr int kPer = 4, kBytes = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  __device__ static float at(const uint4& v, int k) { return __uint_as_float((&v.x)[k]); }
  __device__ static float one(const char* p) { return *reinterpret_cast<const float*>(p); }
  __device__ static uint32_t raw(const char* p) { return *reinterpret_cast<const uint32_t*>(p); }
  __device__ static void put(uint4& v, int k, const char* p) { (&v.x)[k] = *reinterpret_cast<const uint32_t*>(p); }
  __device__ static float top(const uint4 (&v)[kVecs]) {
    float m = __uint_as_float(v[0].x);
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
      m = max_nan(max_nan(m, __uint_as_float(v[j].x)),
                  max_nan(max_nan(__uint_as_float(v[j].y), __uint_as_float(v[j].z)), __uint_as_float(v[j].w)));
    return m;
  }
  __device__ static void keep(uint4& v, uint32_t bits) {
    v.x = (bits & 1u) ? v.x : kNegInf;
    v.y = (bits & 2u) ? v.y : kNegInf;
    v.z = (bits & 4u) ? v.z : kNegInf;
    v.w = (bits & 8u) ? v.w : kNegInf;
  }
};

template <uint32_t NEG_INF>
struct Half {  // either 16-bit type
  static constexpr int kPer = 8, kBytes = 2;
  static constexpr uint32_t kNegInf = NEG_INF | (NEG_INF << 16);
  __device__ static uint32_t raw(const char* p) { return *reinterpret_cast<const uint16_t*>(p); }
  __device__ static void put(uint4& v, int k, const char* p) {
    uint32_t& w = (&v.x)[k >> 1];
    const uint32_t b = *reinterpret_cast<const uint16_t*>(p);
    w = (k & 1) ? (w & 0x0000ffffu) | (b << 16) : (w & 0xffff0000u) | b;
  }
  // Four bits spread to the top bits of four bytes by one multiplication, then each copied over
  // its half of a pair (prmt's sign mode).
  __device__ static void keep(uint4& v, uint32_t bits) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t spread = ((bits >> (4 * k)) & 15u) * 0x10204080u;
      uint32_t low, high;
      asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(low) : "r"(spread));
      asm("prmt.b32 %0, %1, 0, 0xbbaa;" : "=r"(high) : "r"(spread));
      (&v.x)[2 * k] = ((&v.x)[2 * k] & low) | (kNegInf & ~low);
      (&v.x)[2 * k + 1] = ((&v.x)[2 * k + 1] & high) | (kNegInf & ~high);
    }
  }
};
struct BF16 : Half<0xff80u> {
  __device__ static float at(const uint4& v, int k) {
    const uint32_t w = (&v.x)[k >> 1];
    return __uint_as_float((k & 1) ? w & 0xffff0000u : w << 16);
  }
  __device__ static float one(const char* p) {
    return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
  }
  __device__ static float top(const uint4 (&v)[kVecs]) {
    const auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h(v[0].x), h(v[0].y)), __hmax2_nan(h(v[0].z), h(v[0].w)));
#pragma unroll
    for (int j = 1; j < kVecs; ++j)
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(h(v[j].x), h(v[j].y)), __hmax2_nan(h(v[j].z), h(v[j].w))));
    return max_nan(__low2float(m), __high2float(m));
  }
};
struct F16 : Half<0xfc00u> {
  __device__ static float at(const uint4& v, int k) {
    const uint32_t w = (&v.x)[k >> 1];
    return __half2float(__ushort_as_half(static_cast<unsigned short>((k & 1) ? w >> 16 : w & 0xffffu)));
  }
  __device__ static float one(const char* p) {
    return __half2float(__ushort_as_half(*reinterpret_cast<const unsigned short*>(p)));
  }
  __device__ static float top(const uint4 (&v)[kVecs]) {
    const auto h = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
    __half2 m = __hmax2_nan(__hmax2_nan(h(v[0].x), h(v[0].y)), __hmax2_nan(h(v[0].z), h(v[0].w)));
#pragma unroll
    for (int j = 1; j < kVecs; ++j)
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(h(v[j].x), h(v[j].y)), __hmax2_nan(h(v[j].z), h(v[j].w))));
    return max_nan(__low2float(m), __high2float(m));
  }
};

// A row's mask: words base[w] | delta[w], or every token (both null).
struct RowMask {
  const uint32_t* base;
  const uint32_t* delta;
  __device__ bool all() const { return base == nullptr && delta == nullptr; }
  __device__ uint32_t word(int32_t w) const { return (base ? __ldg(base + w) : 0u) | (delta ? delta[w] : 0u); }
  // bits of the n <= 8 tokens from t0 on, of which those outside [0, vocab) are 0
  __device__ uint32_t bits(int32_t t0, int32_t n, int32_t vocab) const {
    uint32_t inside = (1u << n) - 1u;
    if (t0 < 0) inside &= kFull << -t0;
    if (t0 + n > vocab) inside &= vocab > t0 ? (1u << (vocab - t0)) - 1u : 0u;
    if (all() || inside == 0u) return inside;
    const int32_t from = t0 < 0 ? 0 : t0, w = from >> 5, last = (vocab - 1) >> 5;
    uint64_t x = word(w);
    if ((from & 31) + n > 32 && w < last) x |= static_cast<uint64_t>(word(w + 1)) << 32;
    const uint32_t got = static_cast<uint32_t>(x >> (from & 31));
    return (t0 < 0 ? got << -t0 : got) & inside;
  }
};

__device__ __forceinline__ RowMask row_mask(const RowMasks& m, int32_t row) {
  if (m.slots) {
    const int32_t slot = m.slots[row];
    if (slot < 0 || slot >= m.max_slots || !m.active[slot]) return RowMask{nullptr, nullptr};
    return RowMask{m.base[slot], m.delta[slot]};
  }
  return RowMask{m.words ? m.words + row * m.stride : nullptr, nullptr};
}

// What the scan leaves for the merge: per (row, share) the sum's parts, and its best keys, best
// first (rising(logit) << 32 | ~token; 0: none).
struct Part {
  double sum;      // of 2^(x kLog2eHi - anchor)
  double far_sum;  // of exp(x - far), from steps whose maximum is far from 0
  float anchor;    // a whole number; -inf: no sum
  float far;       // -inf: no far sum
};

struct ScanArgs {
  SelectArgs a;
  Part* parts;      // [rows][shares]
  uint64_t* keys;   // [rows][shares][candidates]
  int32_t shares, steps_per_share;
  int32_t pool;     // beams * shares * candidates
};

__device__ __forceinline__ uint64_t make_key(uint32_t order, int32_t token) {
  return (static_cast<uint64_t>(order) << 32) | static_cast<uint32_t>(~token);
}

// Out of line: a launch's first CTAs wait for every instruction that they reach.
__device__ __noinline__ double exp_apart(double x) { return exp(x); }
__device__ __noinline__ uint32_t mask_bits(const RowMask mask, int32_t t0, int32_t n, int32_t vocab) {
  return mask.bits(t0, n, vocab);
}

// 2^k of a whole number k <= 0 (0 below the normal doubles), exactly.
__device__ __forceinline__ double power2(float k) {
  return k < -1000.0f ? 0.0 : __hiloint2double((1023 + static_cast<int32_t>(k)) << 20, 0);
}

// Row r takes part: its score is finite and the beam has not ended.
__device__ __forceinline__ bool row_scans(const SelectArgs& a, int32_t row) {
  const bool ended = a.finished && a.finished[row];
  return isfinite(a.scores[row]) && !ended;
}

struct ScanShared {
  uint4 ring[kSteps * kVecs * kScanThreads];  // afterwards the listed entries' vectors
  union {
    uint32_t tops[kRound][kScanThreads];  // rising() of each thread's maximum in each step
    uint64_t pushed[kPushCap];            // afterwards the listed entries' keys
  };
  alignas(16) uint64_t few[kRankMost];
  int32_t list[kListCap];              // entries: step of the round * kScanThreads + thread
  uint32_t thread_top[kScanWarps][32];  // the threads' maxima in the round
  uint32_t warp_bound[2][kScanWarps];
  Part warp_part[kScanWarps];
  int32_t counts[2][kScanWarps];
  int32_t listed, count, few_count;
};
static_assert(kListCap * kVecs <= kSteps * kVecs * kScanThreads, "the ring holds the listed vectors");

__device__ __forceinline__ int32_t block_total(int32_t mine, int32_t (&counts)[kScanWarps]) {
  const int32_t of_warp = __reduce_add_sync(kFull, mine);
  if ((threadIdx.x & 31) == 0) counts[threadIdx.x >> 5] = of_warp;
  __syncthreads();
  int32_t total = 0;
#pragma unroll
  for (int32_t w = 0; w < kScanWarps; ++w) total += counts[w];
  return total;
}

__device__ __forceinline__ uint32_t block_most(uint32_t mine, int32_t (&counts)[kScanWarps]) {
  const uint32_t of_warp = __reduce_max_sync(kFull, mine);
  __syncthreads();  // whoever used the counts before has read them
  if ((threadIdx.x & 31) == 0) counts[threadIdx.x >> 5] = static_cast<int32_t>(of_warp);
  __syncthreads();
  uint32_t most = 0;
#pragma unroll
  for (int32_t w = 0; w < kScanWarps; ++w) most = max(most, static_cast<uint32_t>(counts[w]));
  return most;
}

// Where a bisection between two orders starts: the bits that both have, the others 0 (all of them,
// if the two are equal).
__device__ __forceinline__ uint32_t above_common(uint32_t bound, uint32_t most) {
  return bound == most ? most : most & ~((2u << (31 - __clz(bound ^ most))) - 1u);
}

// At most kRankMost of the n keys in sh.pushed, `wanted` best among them: the keys are bisected
// until few are above the edge.  Returns how many are left.
__device__ __noinline__ int32_t fewer_keys(ScanShared& sh, int32_t n, int32_t wanted) {
  const int32_t tid = threadIdx.x;
  constexpr int32_t kEach = kPushCap / kScanThreads;
  uint64_t key[kEach], edge = 0;
#pragma unroll
  for (int32_t i = 0; i < kEach; ++i) key[i] = tid + i * kScanThreads < n ? sh.pushed[tid + i * kScanThreads] : 0u;
  int32_t turn = 0;
#pragma unroll 1
  for (int32_t bit = 63; bit >= 0; --bit, turn ^= 1) {
    const uint64_t trial = edge | (1ull << bit);
    int32_t mine = 0;
#pragma unroll
    for (int32_t i = 0; i < kEach; ++i) mine += key[i] >= trial;
    const int32_t total = block_total(mine, sh.counts[turn]);
    if (total >= wanted) {
      edge = trial;
      if (total <= kRankMost) break;
    }
  }
  __syncthreads();
  if (tid == 0) sh.few_count = 0;
  __syncthreads();
#pragma unroll
  for (int32_t i = 0; i < kEach; ++i)
    if (key[i] >= edge && key[i] != 0u) sh.pushed[atomicAdd(&sh.few_count, 1)] = key[i];
  __syncthreads();
  return sh.few_count;
}

// The best min(n, wanted) of the n keys in sh.pushed, in order, into sh.few (all threads; a
// barrier before the call has made the keys visible and one is passed after them).
__device__ __forceinline__ int32_t best_of(ScanShared& sh, int32_t n, int32_t wanted) {
  if (n > kRankMost) n = fewer_keys(sh, n, wanted);
  // several threads of a warp share a key's comparisons
  int32_t split = 1;
  while (split < 32 && n * split * 2 <= kScanThreads) split <<= 1;
  const int32_t i = threadIdx.x / split;
  const uint64_t mine = i < n ? sh.pushed[i] : 0u;
  int32_t rank = 0;
#pragma unroll 4
  for (int32_t j = threadIdx.x & (split - 1); j < n; j += split) rank += sh.pushed[j] > mine;
#pragma unroll 1
  for (int32_t d = 1; d < split; d <<= 1) rank += __shfl_xor_sync(kFull, rank, d);
  if (i < n && rank < wanted) sh.few[rank] = mine;  // the same from each of them
  __syncthreads();
  return min(n, wanted);
}

// Where an entry's vector j begins: entry = step of the round * kScanThreads + thread, and
// `first` the token of the round's first vector (a warp's vectors of a step are consecutive).
template <typename E>
__device__ __forceinline__ int32_t vector_token(int32_t entry, int32_t j, int32_t first) {
  const int32_t step = entry / kScanThreads, thread = entry % kScanThreads;
  return first + (((step * kScanWarps + thread / 32) * kVecs + j) * 32 + thread % 32) * E::kPer;
}

// More than kListCap entries reach the bound (ties, or fewer than `wanted` threads saw a token):
// the bound rises by bisection until at most kRankMost do.  Where equal maxima do not let it,
// the entries above it are taken and, of those at it, the ones of the earliest steps that hold
// `wanted` together: a later step's equal tokens come after theirs.  That is fewer than
// 2 * wanted + kScanThreads <= kListCap entries.  Returns the bound.
__device__ __noinline__ uint32_t list_crowded(ScanShared& sh, uint32_t bound, int32_t steps, int32_t wanted) {
  const int32_t tid = threadIdx.x;
  int32_t turn = 0;
  const auto count_if = [&](auto pick) {
    int32_t mine = 0;
#pragma unroll 1
    for (int32_t step = 0; step < steps; ++step) mine += pick(sh.tops[step][tid], step);
    turn ^= 1;
    return block_total(mine, sh.counts[turn]);
  };
  int32_t level = 0x7fffffff, last = kRound;  // entries at the edge are taken up to step `last`
  uint32_t most = 0;
  for (int32_t step = 0; step < steps; ++step) most = max(most, sh.tops[step][tid]);
  most = block_most(most, sh.counts[0]);
  uint32_t edge = above_common(bound, most);
  for (int32_t bit = 31 - __clz(bound ^ most); bit >= 0 && level > kRankMost; --bit) {
    const uint32_t trial = edge | (1u << bit);
    const int32_t total = count_if([=](uint32_t o, int32_t) { return o >= trial; });
    if (total >= wanted) {
      edge = trial;
      level = total;
    }
  }
  if (level > kRankMost) {
    const int32_t above = count_if([=](uint32_t o, int32_t) { return o > edge; });
    for (last = 0; last < steps; ++last)
      if (count_if([=](uint32_t o, int32_t step) { return o == edge && step <= last; }) >= wanted - above) break;
  }
  edge = max(edge, kRisingLowest);
  __syncthreads();
  if (tid == 0) sh.listed = 0;
  __syncthreads();
#pragma unroll 1
  for (int32_t step = 0; step < steps; ++step) {
    const uint32_t o = sh.tops[step][tid];
    if (o >= edge && (o > edge || step <= last)) {
      const int32_t n = atomicAdd(&sh.listed, 1);
      if (n < kListCap) sh.list[n] = step * kScanThreads + tid;
    }
  }
  __syncthreads();
  return edge;
}

// Too many tokens of the vectors in sh.ring reach the bound: it rises by bisection until at
// most kRankMost do, and where equal logits do not let it, the lowest tokens are taken.  Their
// keys, `wanted` to kRankMost, follow the `held` ones in sh.pushed.
template <typename E>
__device__ __noinline__ void push_crowded(ScanShared& sh, uint32_t bound, int32_t vectors, int32_t first, int32_t held,
                                          int32_t wanted) {
  constexpr int32_t kPer = E::kPer;
  const int32_t tid = threadIdx.x;
  int32_t turn = 0;
  const auto count_if = [&](auto pick) {
    int32_t mine = 0;
#pragma unroll 1
    for (int32_t i = tid; i < vectors; i += kScanThreads) {
      const uint4 v = sh.ring[i];
      const int32_t t0 = vector_token<E>(sh.list[i / kVecs], i % kVecs, first);
#pragma unroll
      for (int32_t k = 0; k < kPer; ++k) mine += pick(rising(E::at(v, k) + 0.0f), t0 + k);
    }
    turn ^= 1;
    return block_total(mine, sh.counts[turn]);
  };
  int32_t level = 0x7fffffff, last = 0x7fffffff;  // of the tokens equal to the edge, those up to `last`
  uint32_t most = 0;
#pragma unroll 1
  for (int32_t i = tid; i < vectors; i += kScanThreads) {
    const uint4 v = sh.ring[i];
#pragma unroll
    for (int32_t k = 0; k < kPer; ++k) most = max(most, rising(E::at(v, k) + 0.0f));
  }
  most = block_most(most, sh.counts[0]);
  uint32_t edge = above_common(bound, most);
  for (int32_t bit = 31 - __clz(bound ^ most); bit >= 0 && level > kRankMost; --bit) {
    const uint32_t trial = edge | (1u << bit);
    const int32_t total = count_if([=](uint32_t o, int32_t) { return o >= trial; });
    if (total >= wanted) {
      edge = trial;
      level = total;
    }
  }
  if (level > kRankMost) {
    const int32_t above = count_if([=](uint32_t o, int32_t) { return o > edge; });
    // the lowest tokens at the edge, by bisection over the listed steps' tokens
    int32_t low = 0x7fffffff, high = 0;
#pragma unroll 1
    for (int32_t i = tid; i < vectors; i += kScanThreads) {
      const int32_t t0 = vector_token<E>(sh.list[i / kVecs], i % kVecs, first);
      low = min(low, t0);
      high = max(high, t0 + kPer);
    }
    low = static_cast<int32_t>(0x7fffffffu - block_most(0x7fffffffu - static_cast<uint32_t>(low), sh.counts[0]));
    high = static_cast<int32_t>(block_most(static_cast<uint32_t>(high), sh.counts[1]));
    turn = 1;
    last = low - 1;  // too few up to here
    for (int32_t bit = 31 - __clz(high - low + 1); bit >= 0; --bit) {
      const int32_t trial = last + (1 << bit);
      if (count_if([=](uint32_t o, int32_t t) { return o == edge && t <= trial; }) < wanted - above) last = trial;
    }
    ++last;
  }
  edge = max(edge, kRisingLowest);
  __syncthreads();
  if (tid == 0) sh.count = held;
  __syncthreads();
#pragma unroll 1
  for (int32_t i = tid; i < vectors; i += kScanThreads) {
    const uint4 v = sh.ring[i];
    const int32_t t0 = vector_token<E>(sh.list[i / kVecs], i % kVecs, first);
#pragma unroll
    for (int32_t k = 0; k < kPer; ++k) {
      const uint32_t o = rising(E::at(v, k) + 0.0f);
      if (o >= edge && (o > edge || t0 + k <= last)) {
        const int32_t n = atomicAdd(&sh.count, 1);
        if (n < kPushCap) sh.pushed[n] = make_key(o, t0 + k);
      }
    }
  }
  __syncthreads();
}

// The parts of a warp's first `width` lanes (a power of two; the others hold none) as one, in
// those lanes.
__device__ __forceinline__ Part total_part(Part p, int32_t width) {
  const float anchor = from_rising(__reduce_max_sync(kFull, rising(p.anchor)));
  double sum = p.anchor == -CUDART_INF_F ? 0.0 : p.sum * power2(p.anchor - anchor);
#pragma unroll 1
  for (int32_t d = 1; d < width; d <<= 1) sum += __shfl_xor_sync(kFull, sum, d);
  float far = p.far;
  double far_sum = 0.0;
  if (__any_sync(kFull, far != -CUDART_INF_F)) {
    far = from_rising(__reduce_max_sync(kFull, rising(far)));
    if (p.far != -CUDART_INF_F) far_sum = p.far_sum * exp_apart(static_cast<double>(p.far) - static_cast<double>(far));
#pragma unroll 1
    for (int32_t d = 1; d < width; d <<= 1) far_sum += __shfl_xor_sync(kFull, far_sum, d);
  }
  return Part{sum, far_sum, anchor, far};
}

__device__ __forceinline__ void copy_async(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared))),
               "l"(global)
               : "memory");
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_async() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A vector that crosses an end of its row: tokens t0 .. t0 + kPer, -inf outside [0, vocab).
template <typename E>
__device__ __noinline__ uint4 load_edge(const char* logits, int32_t t0, int32_t vocab) {
  uint4 v = make_uint4(E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf);
#pragma unroll
  for (int32_t k = 0; k < E::kPer; ++k)
    if (t0 + k >= 0 && t0 + k < vocab) E::put(v, k, logits + static_cast<int64_t>(t0 + k) * E::kBytes);
  return v;
}
template <typename E>
__device__ __forceinline__ uint4 load_vector(const char* logits, int32_t t0, int32_t vocab) {
  if (t0 >= 0 && t0 + E::kPer <= vocab) return *reinterpret_cast<const uint4*>(logits + static_cast<int64_t>(t0) * E::kBytes);
  return load_edge<E>(logits, t0, vocab);
}

template <typename E, bool MASKED, bool RENORMALIZE>
__global__ void __launch_bounds__(kScanThreads, 4) scan_kernel(const __grid_constant__ ScanArgs s) {
  extern __shared__ __align__(16) char dynamic[];
  ScanShared& sh = *reinterpret_cast<ScanShared*>(dynamic);
  asm volatile("griddepcontrol.wait;" ::: "memory");               // what came before on the stream is complete
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge waits for this grid's end
  constexpr int32_t kPer = E::kPer;
  constexpr int32_t kWarpTokens = 32 * kVecs * kPer;  // a warp's vectors of a step are consecutive
  constexpr int32_t kStepTokens = kScanWarps * kWarpTokens;
  constexpr uint32_t kAll = (1u << kPer) - 1u;
  constexpr bool kSkips = MASKED && RENORMALIZE;  // vectors without an allowed token are not read
  static_assert(kRound % 8 == 0, "mask words are loaded eight steps at a time");
  static_assert(kVecs * kPer <= 32, "a lane's bits of a step fit one word");
  const SelectArgs& a = s.a;
  const int32_t row = blockIdx.x / s.shares, share = blockIdx.x - row * s.shares;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t wanted = a.candidates, vocab = a.vocab;
  const bool scans = row_scans(a, row);
  const char* logits = a.logits + static_cast<int64_t>(row) * a.row_stride * E::kBytes;
  // vectors start at 16-byte boundaries, so the first may begin before the row
  const int32_t head = static_cast<int32_t>(reinterpret_cast<uintptr_t>(logits) & 15u) / E::kBytes;
  const int32_t begin = share * s.steps_per_share;
  const int32_t end = min(begin + s.steps_per_share, (vocab + head + kStepTokens - 1) / kStepTokens);

  // the warp's first token of a step; a lane's vectors follow one another at 32 vectors' distance
  const auto warp_token = [&](int32_t step) { return step * kStepTokens + warp * kWarpTokens - head; };
  const RowMask mask = MASKED ? row_mask(a.masks, row) : RowMask{nullptr, nullptr};
  // The mask words that the lanes hold of the warp's tokens, `kWords` steps from `step` on
  // (aligned rows; tokens past the row cleared), into the table, where the steps' maxima will lie.
  // The loads come before the first store: a store waits for its own load.
  constexpr int32_t kWords = 8;
  const auto load_words = [&](int32_t step, int32_t stop, uint32_t* to) {
    uint32_t got[kWords];
    const int32_t w0 = (step * kStepTokens + warp * kWarpTokens) / 32 + lane;
    const int32_t steps = lane * 32 < kWarpTokens ? stop - step : 0;
    const uint32_t* words = mask.base ? mask.base : mask.delta;
    const uint32_t* more = mask.base ? mask.delta : nullptr;
#pragma unroll
    for (int32_t k = 0; k < kWords; ++k) {
      const int32_t w = w0 + k * (kStepTokens / 32);
      got[k] = k < steps && w * 32 < vocab ? words ? words[w] : kFull : 0u;
    }
    if (more) {
#pragma unroll
      for (int32_t k = 0; k < kWords; ++k) {
        const int32_t w = w0 + k * (kStepTokens / 32);
        if (k < steps && w * 32 < vocab) got[k] |= more[w];
      }
    }
#pragma unroll
    for (int32_t k = 0; k < kWords; ++k) {
      const int32_t left = vocab - (w0 + k * (kStepTokens / 32)) * 32;
      to[k * kScanThreads] = left > 0 && left < 32 ? got[k] & ((1u << left) - 1u) : got[k];
    }
  };
  // from the lanes' words each lane's own bits, kPer a vector
  const auto own_bits = [&](int32_t step, uint32_t word) {
    uint32_t bits = 0u;
    if (head == 0) {
      if (!__any_sync(kFull, word != 0u)) return 0u;
      constexpr uint32_t kEvery = kVecs * kPer == 32 ? kFull : (1u << (kVecs * kPer & 31)) - 1u;
      if (__all_sync(kFull, word == kFull || lane * 32 >= kWarpTokens)) return kEvery;
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j) {
        const uint32_t got = __shfl_sync(kFull, word, j * kPer + lane * kPer / 32);
        bits |= ((got >> ((lane * kPer) & 31)) & kAll) << (j * kPer);
      }
    } else if (step < end) {
#pragma unroll 1
      for (int32_t j = 0; j < kVecs; ++j) {
        const int32_t t0 = warp_token(step) + (j * 32 + lane) * kPer;
        if (t0 < vocab) bits |= mask_bits(mask, t0, kPer, vocab) << (j * kPer);
      }
    }
    return bits;
  };
  // the loads of a step into the ring (`to`: the thread's first slot)
  const auto issue = [&](int32_t step, uint32_t bits, uint4* to) {
    const int32_t t0 = warp_token(step);
    if (t0 >= 0 && t0 + kWarpTokens <= vocab) {  // uniform in the warp
      const char* from = logits + static_cast<int64_t>(t0) * E::kBytes + lane * 16;
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j) {
        if (!kSkips || ((bits >> (j * kPer)) & kAll))
          copy_async(to + j * kScanThreads, from + j * 512);
        else
          to[j * kScanThreads] = make_uint4(E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf);
      }
    } else {
#pragma unroll 1
      for (int32_t j = 0; j < kVecs; ++j) {
        const int32_t t = t0 + (j * 32 + lane) * kPer;
        if (t < vocab && (!kSkips || ((bits >> (j * kPer)) & kAll)))
          to[j * kScanThreads] = load_vector<E>(logits, t, vocab);
        else
          to[j * kScanThreads] = make_uint4(E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf);
      }
    }
  };

  double sum = 0.0, far_sum = 0.0;  // this thread's, relative to the warp's anchor and far
  float anchor = -CUDART_INF_F, far = -CUDART_INF_F;
  float limit = -CUDART_INF_F;      // logits above it raise the anchor
  int32_t held = 0;                 // best keys of earlier rounds, in sh.few

#pragma unroll 1
  for (int32_t round = begin; round < end; round += kRound) {
    const int32_t stop = min(round + kRound, end);
    uint32_t bits[kSteps] = {0u, 0u};
    if (MASKED) {
      if (!scans) return;
      if (head == 0) {
#pragma unroll 1
        for (int32_t k = 0; k < kRound && round + k < stop; k += kWords) load_words(round + k, stop, &sh.tops[k][tid]);
      }
      bits[0] = own_bits(round, sh.tops[0][tid]);
      if (round + 1 < stop) bits[1] = own_bits(round + 1, sh.tops[1][tid]);
    }
#pragma unroll 1
    for (int32_t k = 0; k < kSteps; ++k) {
      if (round + k < stop) issue(round + k, k ? bits[1] : bits[0], sh.ring + k * kVecs * kScanThreads + tid);
      commit_async();
    }
    if (!MASKED && !scans) {  // the first loads did not wait for the row's flags
      wait_async<0>();
      return;
    }
    float best = -CUDART_INF_F;  // the thread's best logit that it may take
#pragma unroll 1
    for (int32_t step = round; step < stop; ++step) {
      wait_async<kSteps - 1>();
      const int32_t at = step - round;
      uint4* slot = sh.ring + (at & 1) * kVecs * kScanThreads + tid;
      const uint32_t own = MASKED ? bits[0] : 0u;
      constexpr uint32_t kEvery = kVecs * kPer == 32 ? kFull : (1u << (kVecs * kPer & 31)) - 1u;
      const bool whole = !MASKED || __all_sync(kFull, own == kEvery);  // the warp's every token is allowed
      const auto next_step = [&]() {  // the slots are read: the step after the next
        if (MASKED) bits[0] = bits[1];
        if (step + 2 < stop) {
          if (MASKED) bits[1] = own_bits(step + 2, sh.tops[at + 2][tid]);
          issue(step + 2, bits[1], slot);
        }
        commit_async();
      };
      if (kSkips && !__any_sync(kFull, own != 0u)) {  // none of the warp's tokens is
        sh.tops[at][tid] = kRisingLowest - 1u;
        next_step();
        continue;
      }
      uint4 v[kVecs];
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j) v[j] = slot[j * kScanThreads];
      if (kSkips && !whole) {
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j) E::keep(v[j], (own >> (j * kPer)) & kAll);
      }
      float shown = E::top(v);
      bool far_step = false;
      if (__any_sync(kFull, !(shown <= limit))) {  // the first tokens, or a new maximum, or a NaN
        const float most = from_rising(__reduce_max_sync(kFull, rising(shown)));
        if (!isfinite(most)) {
          if (anchor == -CUDART_INF_F) anchor = 0.0f;  // whatever the anchor, the sum will show it
        } else if (fabsf(most) < kFar) {
          const float near = ceilf(most * kLog2eHi) - kAbove;
          if (near > anchor) {
            sum = anchor == -CUDART_INF_F ? 0.0 : sum * power2(anchor - near);
            anchor = near;
            limit = (near + kAbove) * 0.693147f;
          }
        } else {
          far_step = true;
        }
      }
      if (far_step) {  // so far from 0 that log2 e's rounding would show: the difference comes first
        const float most = from_rising(__reduce_max_sync(kFull, rising(shown)));
        double part = 0.0;
#pragma unroll 1
        for (int32_t j = 0; j < kVecs; ++j) {
          uint4 x = slot[j * kScanThreads];
          if (kSkips) E::keep(x, (own >> (j * kPer)) & kAll);
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int32_t k = 0; k < kPer; ++k) {
            const float d = E::at(x, k) - most;
            acc[k & 3] += exp2_fast(fmaf(d, kLog2eHi, d * kLog2eLo));
          }
          part += static_cast<double>((acc[0] + acc[1]) + (acc[2] + acc[3]));
        }
        const float higher = fmaxf(far, most);
        far_sum = (far == -CUDART_INF_F ? 0.0 : far_sum * exp_apart(static_cast<double>(far) - static_cast<double>(higher))) +
                  part * exp_apart(static_cast<double>(most) - static_cast<double>(higher));
        far = higher;
      } else if (anchor != -CUDART_INF_F) {
        // exp(x) as 2^(x kLog2eHi - anchor) with a whole anchor near the maximum: sums of
        // different anchors differ by exact powers of two.  Five additions deep (see kNear).
        const uint64_t hi = pack2(kLog2eHi, kLog2eHi), back = pack2(-anchor, -anchor);
        uint64_t acc[2] = {0, 0};
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j) {
          if (kSkips && !whole && !__any_sync(kFull, (own >> (j * kPer)) & kAll)) continue;
          uint64_t e[kPer / 2];
#pragma unroll
          for (int32_t k = 0; k < kPer; k += 2) {
            const uint64_t y = fma2(pack2(E::at(v[j], k), E::at(v[j], k + 1)), hi, back);
            e[k >> 1] = pack2(exp2_fast(low(y)), exp2_fast(high(y)));
          }
#pragma unroll
          for (int32_t n = kPer / 4; n > 0; n >>= 1)
#pragma unroll
            for (int32_t k = 0; k < n; ++k) e[k] = add2(e[k], e[k + n]);
          acc[j & 1] = add2(acc[j & 1], e[0]);
        }
        const uint64_t all = add2(acc[0], acc[1]);
        sum += static_cast<double>(low(all) + high(all));
      }
      if (MASKED && !RENORMALIZE && !whole) {
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j) E::keep(v[j], (own >> (j * kPer)) & kAll);
        shown = E::top(v);
      }
      sh.tops[at][tid] = rising(shown + 0.0f);
      best = fmaxf(best, shown);
      next_step();
    }

    // the best tokens of the round and of the keys held: the entries that reach a bound which
    // `wanted` tokens reach -- the least, over the warps, of a warp's (wanted / 8)-th best thread,
    // or one warp's own wanted-th best, whichever is more -- and, once enough keys are held, more
    // than the last of them
    const int32_t steps = stop - round;
    const int32_t first = round * kStepTokens - head;
    {
      const uint32_t mine = rising(best + 0.0f);
      sh.thread_top[warp][lane] = mine;
      __syncwarp();
      int32_t rank = 0;
#pragma unroll
      for (int32_t k = 0; k < 8; ++k) {
        const uint4 other = reinterpret_cast<const uint4*>(sh.thread_top[warp])[k];
        rank += (other.x > mine) + (other.y > mine) + (other.z > mine) + (other.w > mine);
      }
      rank += __popc(__match_any_sync(kFull, mine) & ((1u << lane) - 1u));  // equal ones by lane
      const uint32_t of_all = __reduce_max_sync(kFull, rank == (wanted + kScanWarps - 1) / kScanWarps - 1 ? mine : 0u);
      const uint32_t of_one = __reduce_max_sync(kFull, rank == wanted - 1 ? mine : 0u);
      if (lane == 0) {
        sh.warp_bound[0][warp] = of_all;
        sh.warp_bound[1][warp] = of_one;
      }
    }
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    uint32_t bound = kFull, alone = 0;
#pragma unroll
    for (int32_t w = 0; w < kScanWarps; ++w) {
      bound = min(bound, sh.warp_bound[0][w]);
      alone = max(alone, sh.warp_bound[1][w]);
    }
    bound = max(bound, alone);
    bound = max(bound, kRisingLowest);
    if (held == wanted) bound = max(bound, static_cast<uint32_t>(sh.few[wanted - 1] >> 32) + 1u);
    if (rising(best + 0.0f) >= bound) {
      uint32_t reached = 0;  // steps
#pragma unroll 4
      for (int32_t at = 0; at < steps; ++at) reached |= sh.tops[at][tid] >= bound ? 1u << at : 0u;
#pragma unroll 1
      for (; reached; reached &= reached - 1u) {
        const int32_t n = atomicAdd(&sh.listed, 1);
        if (n < kListCap) sh.list[n] = (__ffs(reached) - 1) * kScanThreads + tid;
      }
    }
    __syncthreads();
    if (sh.listed > kListCap) bound = max(bound, list_crowded(sh, bound, steps, wanted));
    const int32_t vectors = min(sh.listed, kListCap) * kVecs;
    if (tid < held) sh.pushed[tid] = sh.few[tid];  // the table's memory: every entry has been read
    if (tid == 0) sh.count = held;
    __syncthreads();
    const float least = from_rising(bound);
    bool over = false;
#pragma unroll 1
    for (int32_t i = tid; i < vectors; i += kScanThreads) {
      const int32_t t0 = vector_token<E>(sh.list[i / kVecs], i % kVecs, first);
      uint4 v = make_uint4(E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf);
      if (t0 < vocab) {
        v = load_vector<E>(logits, t0, vocab);
        if (MASKED && !mask.all())
          E::keep(v, head == 0 ? (mask.word(t0 >> 5) >> (t0 & 31)) & kAll : mask_bits(mask, t0, kPer, vocab));
      }
      sh.ring[i] = v;
      uint32_t reached = 0;
#pragma unroll
      for (int32_t k = 0; k < kPer; ++k) reached |= E::at(v, k) >= least ? 1u << k : 0u;
#pragma unroll 1
      for (; reached; reached &= reached - 1u) {
        const int32_t k = __ffs(reached) - 1;
        const float x = E::one(reinterpret_cast<const char*>(sh.ring + i) + k * E::kBytes) + 0.0f;
        const int32_t n = atomicAdd(&sh.count, 1);
        if (n < kPushCap) sh.pushed[n] = make_key(rising(x), t0 + k);
        over |= n >= kPushCap;
      }
    }
    if (__syncthreads_or(over)) push_crowded<E>(sh, bound, vectors, first, held, wanted);
    held = best_of(sh, min(sh.count, kPushCap), wanted);
  }
  if (!scans) return;  // a share past the row's end
#pragma unroll
  for (int32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
  if (far != -CUDART_INF_F) {  // uniform in the warp
#pragma unroll
    for (int32_t d = 16; d > 0; d >>= 1) far_sum += __shfl_xor_sync(kFull, far_sum, d);
  }
  if (lane == 0) sh.warp_part[warp] = Part{sum, far_sum, anchor, far};
  uint64_t* out = s.keys + static_cast<int64_t>(blockIdx.x) * wanted;
#pragma unroll 1
  for (int32_t i = tid; i < wanted; i += kScanThreads) out[i] = i < held ? sh.few[i] : 0u;
  __syncthreads();
  if (warp == 0) {
    Part p = lane < kScanWarps ? sh.warp_part[lane] : Part{0.0, 0.0, -CUDART_INF_F, -CUDART_INF_F};
    p = total_part(p, kScanWarps);
    if (lane == 0) s.parts[blockIdx.x] = p;
  }
}

// ---------------------------------------------------------------------------------------
// Selection, second kernel: one CTA per group scores the rows' candidates in 64 bits and
// orders the best: 4 us of latencies (loads, a logarithm, four barriers) behind a launch that
// overlaps the scan's end.  Above kDirect candidates a histogram of their distances from the best
// leaves few to put in order (a bisection of their bits took 11 us where this takes 7, and a
// sample's bound kept hundreds where beams' scores differ: 26 us).

constexpr int32_t kMergeThreads = 512;
constexpr int32_t kMergeWarps = kMergeThreads / 32;
constexpr int32_t kMergeKeys = 4;    // keys that a thread loads ahead
constexpr int32_t kDirect = 128;     // so many candidates are put in order without a selection before
constexpr int32_t kBuckets = 512;    // of 1/16 of a score's unit each
// Two beams' candidates nearer than this are ordered by log-sums taken again in 64 bits.  A scan's
// log-sum is within 9.8e-7 of the exact one, so the difference of two is within 1.96e-6.  A warp's
// terms are 2^y, y = x kLog2eHi - anchor, whose largest lies in (kAbove - 1, kAbove] = (7, 8] (give
// or take 0.03 by rounding); a sum's relative error is the mean of its terms' errors by weight:
//   3.4e-7  y is rounded once: by 2^-21 at most while |y| < 16, which moves 2^y by 2^-21 ln 2.  A warp
//           takes up to 2^17 tokens (2^20 on 8 warps), so those at y <= -16 weigh 2^17 2^-16 / 2^7 at
//           most and add 1e-8;
//   1.0e-7  log2 e is taken as kLog2eHi, 1.34e-8 of it too small: a term moves by that times |x - ref|
//           (in the natural unit), whose mean by weight is within 10 ln 2: at the upper end y <= 8, at
//           the lower an entropy bounds it, -mean(y) <= log2(2^17) - log2(2^7) = 10;
//   2.4e-7  the exponential, 2^-22 (its documented bound);
//   3.0e-7  five 32-bit additions from a term to the 64-bit sum, 2^-24 each.
// Steps far from zero (kFar) stand below these: their y reaches 0 and not 8, but 2^10 tokens share a
// maximum, x - most is exact wherever it counts, both parts of log2 e are taken and the additions are
// three deep.  Merging is in 64 bits by exact powers of two.
// Random logits bring two beams this near in one call of 60 (32 groups of 16 beams, 32 candidates)
// to 1,600 (8 beams, 8 candidates), whose merge then takes about 40 us a row more.
constexpr double kNear = 2e-6;

struct MergeShared {
  double log_sum[kMaxBeams];   // log of the row's sum of exp(x - ref)
  double ref[kMaxBeams];
  double score[kMaxBeams];
  int32_t state[kMaxBeams];    // 0 offers nothing, 1 candidates, 2 ended, 3 candidates, 64-bit sum
  int32_t again[kMaxBeams];
  int32_t like[kMaxBeams];     // the first beam known to have the same row: what holds of its sum holds of this one's
  uint64_t best[kMaxCandidates];  // rising() of the best scores, and their codes
  uint32_t best_code[kMaxCandidates];
  double warp_sum[kMergeWarps], table[64];
  unsigned long long warp_most[kMergeWarps], warp_least[kMergeWarps];
  uint32_t warp_top[kMergeWarps];
  int32_t counts[2][kMergeWarps];
  int32_t bucket[kBuckets];          // candidates by their distance from the best
  int32_t count;
};

// exp(x) in 64 bits for x up to 700 (below -700, where a sum of 1 or more does not see it, exp(-700)): with k the whole number nearest
// 64 x / ln 2 and r the rest, exp(x) = 2^(k / 64) exp(r), where 2^(j / 64) for j = 0 .. 63 comes
// from a table, exp(r) for |r| <= ln 2 / 128 from its series (the next term is below 2^-54) and the
// whole power of two is added to the exponent (the table-driven method of Tang, ACM TOMS 1989).
// A fifth of the 64-bit operations of a general exp, which is what bounds a row's sum.
constexpr double kLn2Part = 0.693147180559945309417 / 64.0;
constexpr double kLn2PartHi = static_cast<double>(static_cast<float>(kLn2Part));  // 24 bits: its product with k is exact
constexpr double kLn2PartLo = kLn2Part - kLn2PartHi;
__device__ __forceinline__ double table_exp(double x, const double* table) {
  x = fmax(x, -700.0);
  const double k = rint(x * (64.0 / 0.693147180559945309417));
  const double r = fma(-k, kLn2PartLo, fma(-k, kLn2PartHi, x));
  double p = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int32_t n = static_cast<int32_t>(k);
  const double e = p * table[n & 63];
  return __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
}

// Sum over N_r of exp(x - ref) in 64 bits, by the whole CTA; ref is near the row's maximum.
template <typename E>
__device__ __noinline__ double row_sum(const SelectArgs& a, int32_t row, double ref, double (&scratch)[kMergeWarps],
                                       double (&table)[64]) {
  if (threadIdx.x < 64) table[threadIdx.x] = exp2(threadIdx.x / 64.0);
  __syncthreads();
  const char* logits = a.logits + static_cast<int64_t>(row) * a.row_stride * E::kBytes;
  const RowMask mask = a.renormalize ? row_mask(a.masks, row) : RowMask{nullptr, nullptr};
  // each thread the same tokens whatever the row's alignment, so that equal rows have equal sums
  const bool aligned = (reinterpret_cast<uintptr_t>(logits) & 15u) == 0;
  const int32_t vecs = (a.vocab + E::kPer - 1) / E::kPer;
  double sum = 0.0;
#pragma unroll 1
  for (int32_t i = threadIdx.x; i < vecs; i += kMergeThreads) {
    const int32_t t0 = i * E::kPer;
    uint4 v = aligned ? load_vector<E>(logits, t0, a.vocab) : load_edge<E>(logits, t0, a.vocab);
    if (!mask.all()) E::keep(v, mask.word(t0 >> 5) >> (t0 & 31) & ((1u << E::kPer) - 1u));
    double part = 0.0;
#pragma unroll 4  // more of them would take more registers than the kernel has, and slow every call
    for (int32_t k = 0; k < E::kPer; ++k) part += table_exp(static_cast<double>(E::at(v, k)) - ref, table);
    sum += part;
  }
#pragma unroll
  for (int32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll 1
  for (int32_t w = 0; w < kMergeWarps; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

// Two rows hold the same logits and masks bit for bit, so that their sums are equal.
template <typename E>
__device__ __noinline__ bool rows_alike(const SelectArgs& a, int32_t row, int32_t other) {
  const char* p = a.logits + static_cast<int64_t>(row) * a.row_stride * E::kBytes;
  const char* q = a.logits + static_cast<int64_t>(other) * a.row_stride * E::kBytes;
  bool differ = false;
  int32_t t = 0;
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & 15u) == 0) {
#pragma unroll 8
    for (int32_t v = threadIdx.x; v < a.vocab / E::kPer; v += kMergeThreads) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[v], y = reinterpret_cast<const uint4*>(q)[v];
      differ |= x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w;
    }
    t = a.vocab / E::kPer * E::kPer;
  }
#pragma unroll 4
  for (t += threadIdx.x; t < a.vocab; t += kMergeThreads)
    differ |= E::raw(p + static_cast<int64_t>(t) * E::kBytes) != E::raw(q + static_cast<int64_t>(t) * E::kBytes);
  if (a.renormalize) {
    const RowMask m = row_mask(a.masks, row), n = row_mask(a.masks, other);
    if (!m.all() || !n.all())
      for (int32_t w = threadIdx.x; w < (a.vocab + 31) / 32; w += kMergeThreads)
        differ |= (m.all() ? kFull : m.word(w)) != (n.all() ? kFull : n.word(w));
  }
  return !__syncthreads_or(differ);
}

// Doubles as unsigned integers of the same order.
__device__ __forceinline__ uint64_t rising(double x) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x));
  return b ^ (static_cast<uint64_t>(static_cast<int64_t>(b) >> 63) | 0x8000000000000000ull);
}
constexpr uint64_t kRisingNone = 0x000fffffffffffffull;  // rising(-infinity)

__device__ __forceinline__ double from_rising(uint64_t o) {
  return __longlong_as_double(static_cast<long long>(o ^ ((o >> 63) ? 0x8000000000000000ull : ~0ull)));
}

// Which sixteenth below the best a score lies in; the last holds all that are farther.
__device__ __forceinline__ int32_t bucket_of(double score, float best) {
  const float below = (best - __double2float_rn(score)) * 16.0f;
  return below < static_cast<float>(kBuckets - 1) ? static_cast<int32_t>(below) : kBuckets - 1;
}

__device__ __forceinline__ int32_t merge_total(int32_t mine, int32_t (&counts)[kMergeWarps]) {
  const int32_t of_warp = __reduce_add_sync(kFull, mine);
  if ((threadIdx.x & 31) == 0) counts[threadIdx.x >> 5] = of_warp;
  __syncthreads();
  const int32_t lane = threadIdx.x & 31;
  return __reduce_add_sync(kFull, lane < kMergeWarps ? counts[lane] : 0);
}

// The candidates of the pool that may be among the best, into kept / kept_code (sh.count of them):
// those within the fewest sixteenths below the best that hold `wanted`, or, where these are many or
// far from the best, those above an edge raised by bisection over the bits that they differ in
// until few are left, equal scores by beam and token.
__device__ __forceinline__ void keep_best(MergeShared& sh, const uint64_t* order, const uint32_t* code, int32_t pool,
                                       int32_t wanted, uint64_t* kept, uint32_t* kept_code) {
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t most_kept = wanted < 32 ? 64 : 2 * wanted;
  uint64_t most = 0, least = ~0ull;
#pragma unroll 1
  for (int32_t i = tid; i < pool; i += kMergeThreads) {
    const uint64_t o = order[i];
    if (o == kRisingNone) continue;
    most = o > most ? o : most;
    least = o < least ? o : least;
  }
  const uint32_t of_warp = __reduce_max_sync(kFull, most ? rising(__double2float_rn(from_rising(most))) : 0u);
  if (lane == 0) sh.warp_top[warp] = of_warp;
#pragma unroll 1
  for (int32_t i = tid; i < kBuckets; i += kMergeThreads) sh.bucket[i] = 0;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  const float top = from_rising(__reduce_max_sync(kFull, lane < kMergeWarps ? sh.warp_top[lane] : 0u));
#pragma unroll 1
  for (int32_t i = tid; i < pool; i += kMergeThreads)
    if (order[i] != kRisingNone) atomicAdd(&sh.bucket[bucket_of(from_rising(order[i]), top)], 1);
  __syncthreads();
  // which bucket holds the wanted-th: first of 32 sets of buckets, then of that set's
  constexpr int32_t kEach = kBuckets / 32;
  static_assert(kEach == 16, "two steps of 32 and 16");
  int32_t upto = 0;
#pragma unroll
  for (int32_t i = 0; i < kEach; ++i) upto += sh.bucket[lane * kEach + i];
#pragma unroll
  for (int32_t d = 1; d < 32; d <<= 1) {
    const int32_t before = __shfl_up_sync(kFull, upto, d);
    if (lane >= d) upto += before;
  }
  const uint32_t sets = __ballot_sync(kFull, upto >= wanted);
  uint64_t edge = kRisingNone + 1;  // candidates of this order, and with it of a code <= last, and above are kept
  uint32_t last = kFull;
  int32_t farthest = kBuckets;      // and at most this far below the best
  if (sets) {  // else fewer than `wanted` in all: every one of them
    const int32_t set = __ffs(sets) - 1;
    const int32_t before_set = set > 0 ? __shfl_sync(kFull, upto, set > 0 ? set - 1 : 0) : 0;
    int32_t within = before_set + (lane < kEach ? sh.bucket[set * kEach + lane] : 0);
    if (lane > 0) within -= before_set;
#pragma unroll
    for (int32_t d = 1; d < kEach; d <<= 1) {
      const int32_t before = __shfl_up_sync(kFull, within, d);
      if (lane >= d) within += before;
    }
    const int32_t at = __ffs(__ballot_sync(kFull, lane < kEach && within >= wanted)) - 1;
    const int32_t level0 = __shfl_sync(kFull, within, at);
    farthest = set * kEach + at;
    if (level0 > most_kept || farthest == kBuckets - 1) {
      farthest = kBuckets;
#pragma unroll 1
      for (int32_t d = 16; d > 0; d >>= 1) {
        const uint64_t m = __shfl_xor_sync(kFull, most, d), l = __shfl_xor_sync(kFull, least, d);
        most = m > most ? m : most;
        least = l < least ? l : least;
      }
      if (lane == 0) {
        sh.warp_most[warp] = most;
        sh.warp_least[warp] = least;
      }
      __syncthreads();
#pragma unroll 1
      for (int32_t w = 0; w < kMergeWarps; ++w) {
        most = sh.warp_most[w] > most ? sh.warp_most[w] : most;
        least = sh.warp_least[w] < least ? sh.warp_least[w] : least;
      }
      int32_t turn = 0, level = pool;
      if (most > least) {
        const int32_t top_bit = 63 - __clzll(static_cast<long long>(most ^ least));
        uint64_t base = most & ~((2ull << top_bit) - 1ull);
#pragma unroll 1
        for (int32_t bit = top_bit; bit >= 0 && level > most_kept; --bit, turn ^= 1) {
          const uint64_t trial = base | (1ull << bit);
          int32_t mine = 0;
#pragma unroll 1
          for (int32_t i = tid; i < pool; i += kMergeThreads) mine += order[i] >= trial;
          const int32_t total = merge_total(mine, sh.counts[turn]);
          if (total >= wanted) {
            base = trial;
            edge = trial;
            level = total;
          }
        }
      } else {
        edge = most;
      }
      if (level > most_kept) {  // equal scores: by beam and token
        int32_t above = 0, equal = 0;
#pragma unroll 1
        for (int32_t i = tid; i < pool; i += kMergeThreads) {
          above += order[i] > edge;
          equal += order[i] == edge;
        }
        above = merge_total(above, sh.counts[turn]);
        turn ^= 1;
        equal = merge_total(equal, sh.counts[turn]);
        turn ^= 1;
        if (above + equal > most_kept && above < wanted) {
          uint32_t before = kFull;  // codes up to before + 1 are kept
#pragma unroll 1
          for (int32_t bit = 25; bit >= 0; --bit, turn ^= 1) {
            const uint32_t trial = before + (1u << bit);
            int32_t mine = 0;
#pragma unroll 1
            for (int32_t i = tid; i < pool; i += kMergeThreads) mine += order[i] == edge && code[i] <= trial;
            if (merge_total(mine, sh.counts[turn]) < wanted - above) before = trial;
          }
          last = before + 1u;
        }
      }
    }
  }
#pragma unroll 1
  for (int32_t i = tid; i < pool; i += kMergeThreads) {
    const uint64_t o = order[i];
    if (o != kRisingNone && (o > edge || (o == edge && code[i] <= last)) &&
        (farthest == kBuckets || bucket_of(from_rising(o), top) <= farthest)) {
      const int32_t at = atomicAdd(&sh.count, 1);
      kept[at] = o;
      kept_code[at] = code[i];
    }
  }
  __syncthreads();
}

template <typename E>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ ScanArgs s) {
  extern __shared__ __align__(16) char dynamic[];
  __shared__ MergeShared sh;
  const SelectArgs& a = s.a;
  const int32_t pool = s.pool, beams = a.beams, shares = s.shares, wanted = a.candidates;
  uint64_t* order = reinterpret_cast<uint64_t*>(dynamic);        // [pool] rising() of the scores
  uint64_t* kept = order + pool;                                 // [pool] those that may be among the best
  uint32_t* code = reinterpret_cast<uint32_t*>(kept + pool);     // [pool] beam << 20 | token, then the kept ones'
  uint32_t* kept_code = code + pool;
  const int32_t group = blockIdx.x, row0 = group * beams;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t of_beam = shares * wanted;
  const uint64_t* keys = s.keys + static_cast<int64_t>(row0) * of_beam;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the scan is complete

  uint64_t ahead[kMergeKeys];
#pragma unroll
  for (int32_t k = 0; k < kMergeKeys; ++k) {
    const int32_t i = tid + k * kMergeThreads;
    ahead[k] = i < pool ? keys[i] : 0u;
  }
  int32_t width = 1;
  while (width < shares && width < 32) width <<= 1;
#pragma unroll 1
  for (int32_t b = warp; b < beams; b += kMergeWarps) {
    const int32_t row = row0 + b;
    const float score = a.scores[row];
    const bool ended = a.finished && a.finished[row];
    Part p{0.0, 0.0, -CUDART_INF_F, -CUDART_INF_F};
    int32_t state = 0;
    double ref = 0.0, log_sum = 0.0;
    if (isfinite(score)) {
      if (ended) {
        state = 2;
      } else {
        if (lane < shares) p = s.parts[static_cast<int64_t>(row) * shares + lane];
#pragma unroll 1
        for (int32_t c = lane + 32; c < shares; c += 32) {
          const Part q = s.parts[static_cast<int64_t>(row) * shares + c];
          if (q.anchor != -CUDART_INF_F) {
            const float anchor = fmaxf(p.anchor, q.anchor);
            p.sum = (p.anchor == -CUDART_INF_F ? 0.0 : p.sum * power2(p.anchor - anchor)) + q.sum * power2(q.anchor - anchor);
            p.anchor = anchor;
          }
          if (q.far != -CUDART_INF_F) {
            const float far = fmaxf(p.far, q.far);
            p.far_sum = (p.far == -CUDART_INF_F ? 0.0 : p.far_sum * exp_apart(static_cast<double>(p.far) - static_cast<double>(far))) +
                        q.far_sum * exp_apart(static_cast<double>(q.far) - static_cast<double>(far));
            p.far = far;
          }
        }
        p = total_part(p, width);
        double sum = p.sum;
        ref = p.anchor == -CUDART_INF_F ? 0.0 : static_cast<double>(p.anchor) * kAnchorLn;
        if (p.far != -CUDART_INF_F) {
          const double far = static_cast<double>(p.far);
          const double higher = p.anchor == -CUDART_INF_F || far > ref ? far : ref;
          sum = (p.anchor == -CUDART_INF_F ? 0.0 : sum * exp_apart(ref - higher)) + p.far_sum * exp_apart(far - higher);
          ref = higher;
        }
        if (isfinite(sum) && sum > 0.0) {
          state = 1;
          log_sum = log(sum);
        }
      }
    }
    if (lane == 0) {
      sh.score[b] = score;
      sh.state[b] = state;
      sh.ref[b] = ref;
      sh.log_sum[b] = log_sum;
      sh.like[b] = b;
    }
  }
  bool compared = false;
  int32_t filled;
#pragma unroll 1
  for (;;) {
    __syncthreads();
    // every candidate's score
    const auto place = [&](int32_t i, uint64_t key) {
      const int32_t b = i / of_beam, state = sh.state[b];
      uint64_t o = kRisingNone;
      uint32_t token = 0;
      if (state == 2) {
        if (i == b * of_beam && a.end_token >= 0) {
          o = rising(sh.score[b] + 0.0);
          token = a.end_token;
        }
      } else if (state && key) {
        token = ~static_cast<uint32_t>(key);
        const double x = from_rising(static_cast<uint32_t>(key >> 32));
        const double v = sh.score[b] + ((x - sh.ref[b]) - sh.log_sum[b]);
        if (isfinite(__double2float_rn(v))) o = rising(v + 0.0);
      }
      order[i] = o;
      code[i] = (static_cast<uint32_t>(b) << 20) | token;
    };
#pragma unroll
    for (int32_t k = 0; k < kMergeKeys; ++k)
      if (tid + k * kMergeThreads < pool) place(tid + k * kMergeThreads, ahead[k]);
#pragma unroll 1
    for (int32_t i = tid + kMergeKeys * kMergeThreads; i < pool; i += kMergeThreads) place(i, keys[i]);
    if (tid < beams) sh.again[tid] = 0;
    __syncthreads();
    int32_t n = pool, at0 = 0;  // the candidates to put in order: order[at0 ..), code[at0 ..)
    if (pool > kDirect) {
      keep_best(sh, order, code, pool, wanted, kept, kept_code);
      at0 = pool;
      n = sh.count;
    }
    // in order, by counting the better ones; several threads of a warp share an item's comparisons
    int32_t valid = 0;
    int32_t split = 1;
    while (split < 32 && n * split * 2 <= kMergeThreads) split <<= 1;
    const int32_t per_pass = kMergeThreads / split, part = tid & (split - 1);
#pragma unroll 1
    for (int32_t i0 = 0; i0 < n; i0 += per_pass) {  // uniform: the shuffles below take whole warps
      const int32_t i = i0 + tid / split;
      const uint64_t mine = i < n ? order[at0 + i] : 0u;
      const uint32_t own = i < n ? code[at0 + i] : 0u;
      int32_t rank = 0;
      if (mine > kRisingNone) {
#pragma unroll 4
        for (int32_t j = part; j < n; j += split) {
          const uint64_t other = order[at0 + j];
          rank += other > mine;
          if (other == mine) rank += code[at0 + j] < own;
        }
      }
#pragma unroll 1
      for (int32_t d = 1; d < split; d <<= 1) rank += __shfl_xor_sync(kFull, rank, d);
      if (mine > kRisingNone && part == 0) {
        ++valid;
        if (rank < wanted) {
          sh.best[rank] = mine;
          sh.best_code[rank] = own;
        }
      }
    }
    filled = min(merge_total(valid, sh.counts[0]), wanted);
    // beams whose candidates the 32-bit sums cannot order: neighbours among the best, and whatever
    // of another beam lies as near to the last of them
    bool unsure = false;
    const auto doubt = [&](uint32_t b) {
      if (sh.state[b] == 1) {
        sh.again[b] = 1;
        unsure = true;
      }
    };
    if (tid + 1 < filled) {
      const uint32_t p = sh.best_code[tid] >> 20, q = sh.best_code[tid + 1] >> 20;
      if (sh.like[p] != sh.like[q] && from_rising(sh.best[tid]) - from_rising(sh.best[tid + 1]) <= kNear) {
        doubt(p);
        doubt(q);
      }
    }
    if (filled == wanted) {
      const uint64_t last_best = sh.best[wanted - 1];
      const uint64_t lowest = rising(from_rising(last_best) - kNear);
      const uint32_t last_beam = sh.best_code[wanted - 1] >> 20;
#pragma unroll 1
      for (int32_t i = tid; i < pool; i += kMergeThreads)
        if (order[i] >= lowest && order[i] <= last_best && sh.like[code[i] >> 20] != sh.like[last_beam]) {
          doubt(code[i] >> 20);
          doubt(last_beam);
        }
    }
    if (!__syncthreads_or(unsure)) break;
    if (!compared) {
      // equal rows (a padded batch's, a beam given twice) have equal sums: nothing to tell apart
      compared = true;
      bool found = false;
#pragma unroll 1
      for (int32_t b = 1; b < beams; ++b)
#pragma unroll 1
        for (int32_t c = 0; c < b; ++c)
          if (sh.again[b] && sh.again[c] && sh.like[b] == b && sh.like[c] == c && sh.log_sum[b] == sh.log_sum[c] &&
              sh.ref[b] == sh.ref[c] && rows_alike<E>(a, row0 + b, row0 + c)) {
            __syncthreads();
            if (tid == 0) sh.like[b] = c;
            __syncthreads();
            found = true;
          }
      if (found) continue;
    }
#pragma unroll 1
    for (int32_t b = 0; b < beams; ++b) {  // at most once for each beam
      if (!sh.again[b] || sh.state[b] != 1) continue;
      const int32_t first = sh.like[b];
      const double sum = row_sum<E>(a, row0 + first, sh.ref[first], sh.warp_sum, sh.table);
      if (tid < beams && sh.like[tid] == first && sh.state[tid] == 1) {
        sh.log_sum[tid] = log(sum);
        sh.state[tid] = 3;
      }
      __syncthreads();
    }
  }
  if (tid < wanted) {
    const int64_t to = static_cast<int64_t>(group) * wanted + tid;
    float score = -CUDART_INF_F;
    int32_t beam = -1, token = -1;
    bool ended = false;
    if (tid < filled) {
      score = __double2float_rn(from_rising(sh.best[tid]));
      beam = static_cast<int32_t>(sh.best_code[tid] >> 20);
      token = static_cast<int32_t>(sh.best_code[tid] & 0xfffffu);
      ended = token == a.end_token || sh.state[beam] == 2;
    }
    a.out_scores[to] = score;
    a.out_beams[to] = beam;
    a.out_tokens[to] = token;
    if (a.out_finished) a.out_finished[to] = ended;
  }
}

// ---------------------------------------------------------------------------------------
// Reordering.
//
// A thread owns a unit (up to 16 bytes) of every row of a group: it brings the unit of each row
// that is someone's parent into its own slots in shared memory (cp.async), waits for them, then
// stores each moved row's from its parent's slot.  So the move is in place whatever cycles the
// parents form, a parent is read once however many children it has, and rows that stay are not
// touched.  A thread fills its slots with as many units as they hold at a time; the CTAs of an
// SM overlap one's loads with another's stores.
//
// Bound by memory: 963 MB of moves (8 caches of 256 rows, ragged lengths) in 151 us, 97% of the
// copy rate; one request's 48 tensors, 165 MB, in 31 us (81%: a CTA's start, with the read of its
// parents, shows).  Units held in registers took 167 and 79 us (a row's addresses and units a
// thread leave few threads), CTAs that walk all tensors 178 and 56.

constexpr int32_t kMoveThreads = 128;
constexpr int32_t kMoveSlots = 24;    // 16-byte slots of a thread (or one per beam, if more)
constexpr int32_t kMoveTensors = 64;  // descriptors of one launch

struct MoveTensor {
  char* data;
  int64_t row_bytes;          // from row to row
  int64_t stride1, stride2;   // bytes, of the two outer dimensions
  uint32_t size1, size2, size3;  // outer sizes; units of the contiguous run
  uint32_t unit;              // axis 3: units of one position
  int32_t axis;               // which of the three `lengths` counts (0: none, 4: one of size 1)
  int32_t log_bytes;          // unit bytes: 1 << log_bytes
};

struct MoveArgs {
  MoveTensor tensors[kMoveTensors];
  int32_t count, groups, beams, slots;
  int64_t rows;
  const int32_t* parents;
  const int32_t* lengths;
  const int32_t* row_of;
};

// One unit of 1 << LOG bytes into a slot, and out of it.
template <int32_t LOG>
__device__ __forceinline__ void fetch_unit(char* slot, const char* from) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(slot));
  if constexpr (LOG == 4)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else if constexpr (LOG == 3)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
  else if constexpr (LOG == 2)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
  else if constexpr (LOG == 1)
    *reinterpret_cast<uint16_t*>(slot) = *reinterpret_cast<const uint16_t*>(from);
  else
    *slot = *from;
}
template <int32_t LOG>
__device__ __forceinline__ void store_unit(char* to, const char* slot) {
  if constexpr (LOG == 4)
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(slot);
  else if constexpr (LOG == 3)
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(slot);
  else if constexpr (LOG == 2)
    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(slot);
  else if constexpr (LOG == 1)
    *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(slot);
  else
    *to = *slot;
}

// A group's moves: rows to read, and rows to write with the slot that each is written from.
struct Moves {
  int32_t source_row[kMaxBeams], target_row[kMaxBeams], target_slot[kMaxBeams];
  unsigned long long parents;
  int32_t sources, targets;
};

// The CTA's tiles of one tensor: every gridDim.x-th.
// Long runs: a tile is a stretch of one run, so that a thread's units follow at fixed distances.
// Short ones: a thread's units are found one by one among all runs' units.
template <int32_t LOG>
__device__ __forceinline__ void move_tensor(const MoveTensor& t, uint32_t size1, uint32_t size2, uint32_t size3,
                                            const Moves& m, char* slots, int32_t slot_count) {
  constexpr int32_t kSlot = kMoveThreads * 16;  // bytes from slot to slot
  constexpr int32_t kNext = kMoveThreads << LOG;
  const int32_t sources = m.sources, targets = m.targets;
  const uint32_t batch = slot_count / sources;  // units a thread holds at a time
  const uint32_t tile_units = batch * kMoveThreads;
  const uint32_t runs = size1 * size2;
  char* mine = slots + threadIdx.x * 16;
  if (runs == 1 || size3 >= tile_units) {
    const uint32_t of_run = (size3 + tile_units - 1) / tile_units;
    const uint64_t tiles = static_cast<uint64_t>(runs) * of_run;
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const uint32_t run = runs == 1 ? 0u : static_cast<uint32_t>(tile) / of_run;
      const uint32_t unit = static_cast<uint32_t>(tile - static_cast<uint64_t>(run) * of_run) * tile_units + threadIdx.x;
      const int32_t n = unit >= size3 ? 0 : static_cast<int32_t>(min(batch, (size3 - unit + kMoveThreads - 1) / kMoveThreads));
      const uint32_t i1 = run / size2, i2 = run - i1 * size2;
      char* at = t.data + (i1 * t.stride1 + i2 * t.stride2 + (static_cast<int64_t>(unit) << LOG));
      for (int32_t i = 0; i < sources; ++i) {
        const char* from = at + m.source_row[i] * t.row_bytes;
        char* slot = mine + i * kSlot;
#pragma unroll 4
        for (int32_t u = 0; u < n; ++u, from += kNext, slot += sources * kSlot) fetch_unit<LOG>(slot, from);
      }
      commit_async();
      wait_async<0>();
      for (int32_t i = 0; i < targets; ++i) {
        char* to = at + m.target_row[i] * t.row_bytes;
        const char* slot = mine + m.target_slot[i] * kSlot;
#pragma unroll 4
        for (int32_t u = 0; u < n; ++u, to += kNext, slot += sources * kSlot) store_unit<LOG>(to, slot);
      }
    }
  } else {
    const uint64_t units = static_cast<uint64_t>(runs) * size3;
    const uint64_t tiles = (units + tile_units - 1) / tile_units;
    const auto place = [&](uint64_t unit) {
      const uint32_t run = units <= 0xffffffffu ? static_cast<uint32_t>(unit) / size3 : static_cast<uint32_t>(unit / size3);
      const uint32_t in_run = static_cast<uint32_t>(unit - static_cast<uint64_t>(run) * size3);
      const uint32_t i1 = run / size2, i2 = run - i1 * size2;
      return t.data + (i1 * t.stride1 + i2 * t.stride2 + (static_cast<int64_t>(in_run) << LOG));
    };
    for (uint64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const uint64_t unit0 = tile * tile_units + threadIdx.x;
      char* slot = mine;
      for (uint32_t u = 0; u < batch && unit0 + u * kMoveThreads < units; ++u) {
        const char* at = place(unit0 + u * kMoveThreads);
        for (int32_t i = 0; i < sources; ++i, slot += kSlot) fetch_unit<LOG>(slot, at + m.source_row[i] * t.row_bytes);
      }
      commit_async();
      wait_async<0>();
      slot = mine;
      for (uint32_t u = 0; u < batch && unit0 + u * kMoveThreads < units; ++u, slot += sources * kSlot) {
        char* at = place(unit0 + u * kMoveThreads);
        for (int32_t i = 0; i < targets; ++i)
          store_unit<LOG>(at + m.target_row[i] * t.row_bytes, slot + m.target_slot[i] * kSlot);
      }
    }
  }
}

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveArgs a) {
  extern __shared__ __align__(16) char slots[];  // [slot][thread] of 16 bytes
  __shared__ Moves m;
  const int32_t group = blockIdx.y, tid = threadIdx.x;
  if (tid < 32) {
    if (tid == 0) m.parents = 0;
    __syncwarp();
    int32_t n = 0, parent[2], target[2], source[2];
    uint32_t who[2];
#pragma unroll
    for (int32_t h = 0; h < 2; ++h) {
      const int32_t b = tid + 32 * h;
      parent[h] = source[h] = target[h] = -1;
      if (b < a.beams) {
        parent[h] = a.parents[group * a.beams + b];
        if (parent[h] >= 0 && parent[h] < a.beams && parent[h] != b) {
          source[h] = group * a.beams + parent[h];
          target[h] = group * a.beams + b;
          if (a.row_of) {
            source[h] = a.row_of[source[h]];
            target[h] = a.row_of[target[h]];
          }
        }
      }
      const bool valid = source[h] >= 0 && source[h] < a.rows && target[h] >= 0 && target[h] < a.rows && source[h] != target[h];
      who[h] = __ballot_sync(kFull, valid);
      if (valid) atomicOr(&m.parents, 1ull << parent[h]);
    }
    __syncwarp();
    const unsigned long long used = m.parents;
#pragma unroll
    for (int32_t h = 0; h < 2; ++h) {
      if ((who[h] >> tid) & 1u) {
        const int32_t at = n + __popc(who[h] & ((1u << tid) - 1u));
        const int32_t slot = __popcll(used & ((1ull << parent[h]) - 1ull));
        m.target_row[at] = target[h];
        m.target_slot[at] = slot;
        m.source_row[slot] = source[h];  // the same from every child of the parent
      }
      n += __popc(who[h]);
    }
    if (tid == 0) {
      m.targets = n;
      m.sources = __popcll(used);
    }
  }
  const uint32_t length = a.lengths ? static_cast<uint32_t>(max(a.lengths[group], 0)) : 0x7fffffffu;
  __syncthreads();
  if (m.targets == 0) return;
  const MoveTensor& t = a.tensors[blockIdx.z];
  const uint32_t size1 = t.axis == 1 ? min(t.size1, length) : t.size1;
  const uint32_t size2 = t.axis == 2 ? min(t.size2, length) : t.size2;
  const uint32_t size3 =
      t.axis == 3 ? static_cast<uint32_t>(min(static_cast<uint64_t>(t.size3), static_cast<uint64_t>(t.unit) * length))
                  : t.size3;
  if (size1 == 0 || size2 == 0 || size3 == 0 || (t.axis == 4 && length == 0)) return;
  switch (t.log_bytes) {
    case 4: move_tensor<4>(t, size1, size2, size3, m, slots, a.slots); break;
    case 3: move_tensor<3>(t, size1, size2, size3, m, slots, a.slots); break;
    case 2: move_tensor<2>(t, size1, size2, size3, m, slots, a.slots); break;
    case 1: move_tensor<1>(t, size1, size2, size3, m, slots, a.slots); break;
    default: move_tensor<0>(t, size1, size2, size3, m, slots, a.slots); break;
  }
}

// ---------------------------------------------------------------------------------------
// The back-trace.

constexpr int32_t kTraceThreads = 256;
constexpr int32_t kTraceWarps = kTraceThreads / 32;
constexpr int32_t kTraceBytes = 96 * 1024;  // shared memory for a window
constexpr uint8_t kNoBeam = 0xff;

struct TraceArgs {
  const int32_t* tokens;
  int64_t token_step, token_group;
  const int32_t* parents;
  int64_t parent_step, parent_group;
  int32_t steps, groups, beams;
  const int32_t* lengths;
  int32_t pad, window, way_stride, segment, segments, cluster, log_lanes;
  int32_t* out;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint8_t peer_byte(const uint8_t* mine, int32_t rank) {
  uint32_t at, got;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  asm volatile("ld.shared::cluster.u8 %0, [%1];" : "=r"(got) : "r"(at) : "memory");
  return static_cast<uint8_t>(got);
}

// Four bytes, asynchronously.
__device__ __forceinline__ void copy_word_async(void* shared, const void* global) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared))),
               "l"(global)
               : "memory");
}

// A cluster of CTAs per group takes stretches of cluster * window steps, from the last to the
// first; each CTA one window.  A window's tokens and parent maps (as bytes) sit in its shared
// memory, cut into segments that threads walk in parallel from every beam.  The segments' maps
// chained give the window's, the later windows' maps (read from the cluster's other CTAs) the
// beam at the window's end of each last place, and a second walk of the segments every step's
// beam, by which the tokens are picked.  So the walk is 2 * segment + segments + cluster links
// long instead of the steps', and the rest is loads and stores side by side.
//
// Bound by that chain of latencies: 32 groups x 8 beams x 1,024 steps 7.6 us, 64 x 32 x 2,048 (35
// MB with the output) 19.5 us, of which the first loads are 4, the two walks 3 and the cluster's
// waits for its slowest CTA about 4; one CTA a group and one load at a time took 14 and 88.
__global__ void __launch_bounds__(kTraceThreads, 4) trace_kernel(const __grid_constant__ TraceArgs a) {
  extern __shared__ __align__(16) uint8_t shared[];
  const int32_t beams = a.beams, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* text = reinterpret_cast<int32_t*>(shared);        // [window][beams + 1]: rows shifted by a bank each
  uint8_t* maps = shared + a.window * (beams + 1) * 4;       // [window][beams]
  uint8_t* way = maps + a.window * beams;                    // [beams][way_stride]: the beam of each last place
  uint8_t* through = way + beams * a.way_stride;             // [segments][beams]: from a segment's end to before it
  uint8_t* enter = through + a.segments * beams;             // [segments][beams]: the beam at its end, per last place
  uint8_t* whole = enter + a.segments * beams;               // [beams]: from the window's end to before it
  uint8_t* carry = whole + kMaxBeams;                        // [beams]: the beam at the stretch's end, per last place
  uint8_t* peers = carry + kMaxBeams;                        // [cluster][1 << log_lanes]: the windows' maps
  const int32_t group = blockIdx.x / a.cluster, rank = blockIdx.x - group * a.cluster;
  const int32_t length = a.lengths ? min(max(a.lengths[group], 0), a.steps) : a.steps;
  int32_t* out = a.out + static_cast<int64_t>(group) * beams * a.steps;
  // threads by beam: 1 << log_lanes >= beams of them to a step or a segment
  const int32_t k_own = tid & ((1 << a.log_lanes) - 1), s_own = tid >> a.log_lanes, s_next = kTraceThreads >> a.log_lanes;
  const bool has_beam = k_own < beams;
  for (int32_t k = tid; k < beams; k += kTraceThreads) carry[k] = static_cast<uint8_t>(k);
  const int32_t stretch = a.window * a.cluster;
  for (int32_t stop = length; stop > 0; stop -= stretch) {
    // rank 0 the last window of the stretch
    const int32_t end = max(stop - rank * a.window, 0), begin = max(end - a.window, 0), count = end - begin;
    const int32_t segments = (count + a.segment - 1) / a.segment;
    const int32_t* parents = a.parents + begin * a.parent_step + group * a.parent_group + k_own;
    const int32_t* tokens = a.tokens + begin * a.token_step + group * a.token_group + k_own;
    if (has_beam) {
#pragma unroll 8
      for (int32_t t = s_own; t < count; t += s_next) {
        const int32_t p = __ldg(parents + t * a.parent_step);
        copy_word_async(text + t * (beams + 1) + k_own, tokens + t * a.token_step);
        maps[t * beams + k_own] = p >= 0 && p < beams ? static_cast<uint8_t>(p) : kNoBeam;
      }
      commit_async();
    }
    __syncthreads();
    // two segments at a time, so that one's load is in flight while the other's is waited for
    for (int32_t s = s_own; s < segments && has_beam; s += 2 * s_next) {
      const int32_t t0 = s * a.segment, t1 = min(t0 + a.segment, count);
      const int32_t u0 = (s + s_next) * a.segment, u1 = min(u0 + a.segment, count);
      int32_t at = k_own, to = k_own;
      for (int32_t t = t1 - 1, u = u1 - 1; t >= t0 || u >= u0; --t, --u) {
        if (t >= t0 && at != kNoBeam) at = maps[t * beams + at];
        if (u >= u0 && to != kNoBeam) to = maps[u * beams + to];
      }
      through[s * beams + k_own] = static_cast<uint8_t>(at);
      if (u0 < count) through[(s + s_next) * beams + k_own] = static_cast<uint8_t>(to);
    }
    __syncthreads();
    if (tid < beams) {
      int32_t at = tid;
      for (int32_t s = segments - 1; s >= 0 && at != kNoBeam; --s) at = through[s * beams + at];
      whole[tid] = static_cast<uint8_t>(at);
    }
    cluster_sync();
    // the windows' maps of the whole stretch, fetched side by side
    for (int32_t i = tid; i < a.cluster << a.log_lanes; i += kTraceThreads)
      if (has_beam) peers[i] = peer_byte(whole + k_own, i >> a.log_lanes);
    __syncthreads();
    if (tid < beams) {
      int32_t at = carry[tid];
      for (int32_t r = 0; r < rank && at != kNoBeam; ++r) at = peers[(r << a.log_lanes) + at];
      int32_t before = at;  // and on to before the stretch
      for (int32_t r = rank; r < a.cluster && before != kNoBeam; ++r) before = peers[(r << a.log_lanes) + before];
      carry[tid] = static_cast<uint8_t>(before);
      for (int32_t s = segments - 1; s >= 0; --s) {
        enter[s * beams + tid] = static_cast<uint8_t>(at);
        if (at != kNoBeam) at = through[s * beams + at];
      }
    }
    __syncthreads();
    uint8_t* own_way = way + k_own * a.way_stride;
    for (int32_t s = s_own; s < segments && has_beam; s += 2 * s_next) {
      const int32_t t0 = s * a.segment, t1 = min(t0 + a.segment, count);
      const int32_t u0 = (s + s_next) * a.segment, u1 = min(u0 + a.segment, count);
      int32_t at = enter[s * beams + k_own], to = u0 < count ? enter[(s + s_next) * beams + k_own] : kNoBeam;
      for (int32_t t = t1 - 1, u = u1 - 1; t >= t0 || u >= u0; --t, --u) {
        if (t >= t0) {
          own_way[t] = static_cast<uint8_t>(at);
          if (at != kNoBeam) at = maps[t * beams + at];
        }
        if (u >= u0) {
          own_way[u] = static_cast<uint8_t>(to);
          if (to != kNoBeam) to = maps[u * beams + to];
        }
      }
    }
    wait_async<0>();
    cluster_sync();  // the ways and texts are there, and the window's map has been read by the others
    for (int32_t k = warp; k < beams; k += kTraceWarps) {
      int32_t* to = out + static_cast<int64_t>(k) * a.steps + begin;
#pragma unroll 8
      for (int32_t t = lane; t < count; t += 32) {
        const int32_t at = way[k * a.way_stride + t];
        to[t] = at == kNoBeam ? a.pad : text[t * (beams + 1) + at];
      }
    }
    __syncthreads();
  }
  {  // the positions past the end, shared out over the cluster
    const int32_t left = a.steps - length;
    for (int32_t k = rank * kTraceWarps + warp; k < beams; k += a.cluster * kTraceWarps)
      for (int32_t t = lane; t < left; t += 32) out[static_cast<int64_t>(k) * a.steps + length + t] = a.pad;
  }
}

// ---------------------------------------------------------------------------------------
// Host side.

int fail(int code, const std::string& message) { return xg_set_error(code, message.c_str()); }

int cuda_fail(cudaError_t e, const char* what) {
  cudaGetLastError();
  return fail(XG_ECUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

#define XG_BEAM_CUDA(call, what)                       \
  do {                                                 \
    const cudaError_t e_ = (call);                     \
    if (e_ != cudaSuccess) return cuda_fail(e_, what); \
  } while (0)

// Shared memory above the default limit is asked for once per device and kernel.
constexpr int kDevices = 64;

int allow_shared(const void* kernel, int32_t bytes, std::atomic<bool> (&done)[kDevices]) {
  int device = 0;
  XG_BEAM_CUDA(cudaGetDevice(&device), "current device");
  if (device < 0 || device >= kDevices) return fail(XG_EINVAL, "device ordinal out of range");
  if (done[device].load(std::memory_order_acquire)) return XG_OK;
  XG_BEAM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "shared memory limit");
  done[device].store(true, std::memory_order_release);
  return XG_OK;
}

// SM counts, asked for once per device.
int sm_count(int32_t* out) {
  static std::atomic<int> known[kDevices];
  int device = 0;
  XG_BEAM_CUDA(cudaGetDevice(&device), "current device");
  if (device < 0 || device >= kDevices) return fail(XG_EINVAL, "device ordinal out of range");
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    XG_BEAM_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device), "SM count");
    known[device].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return XG_OK;
}

struct Plan {
  int32_t shares, steps_per_share, pool;
  int64_t bytes;
};

int check_sizes(int32_t groups, int32_t beams, int32_t vocab, int32_t dtype, int32_t candidates) {
  if (dtype != XG_F32 && dtype != XG_BF16 && dtype != XG_F16) return fail(XG_EINVAL, "logits must be float32, bfloat16 or float16");
  if (groups < 0 || beams < 1 || beams > kMaxBeams)
    return fail(XG_EINVAL, "a group holds 1 to " + std::to_string(kMaxBeams) + " beams, got " + std::to_string(beams));
  if (candidates < 1 || candidates > kMaxCandidates)
    return fail(XG_EINVAL, "candidates must be between 1 and " + std::to_string(kMaxCandidates) + ", got " +
                               std::to_string(candidates));
  if (vocab < 1 || vocab > kMaxVocab)
    return fail(XG_EINVAL, "the vocabulary must hold 1 to " + std::to_string(kMaxVocab) + " tokens, got " + std::to_string(vocab));
  if (static_cast<int64_t>(groups) * beams > 0x7fffffff / kMaxCandidates) return fail(XG_EINVAL, "too many logits rows");
  return XG_OK;
}

int plan(int32_t groups, int32_t beams, int32_t vocab, int32_t dtype, int32_t candidates, Plan* out) {
  int32_t sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int32_t per = dtype == XG_F32 ? 4 : 8;
  const int32_t step = kScanThreads * kVecs * per;  // a misaligned row's vectors start up to a vector early
  const int32_t tiles = (vocab + per - 1 + step - 1) / step;
  const int64_t rows = static_cast<int64_t>(groups) * beams;
  // one wave of CTAs (four on an SM), but at least two shares of a row unless there are many rows,
  // so that no SM ends with a whole row more than the others
  int64_t shares = rows > 0 ? static_cast<int64_t>(sms) * 4 / rows : 1;
  if (shares < 2 && rows < static_cast<int64_t>(sms) * 8) shares = 2;
  if (shares > kPoolMax / (beams * candidates)) shares = kPoolMax / (beams * candidates);
  if (shares > tiles) shares = tiles;
  if (shares < 1) shares = 1;
  out->steps_per_share = static_cast<int32_t>((tiles + shares - 1) / shares);
  out->shares = (tiles + out->steps_per_share - 1) / out->steps_per_share;
  out->pool = beams * out->shares * candidates;
  out->bytes = rows * out->shares * (static_cast<int64_t>(sizeof(Part)) + candidates * static_cast<int64_t>(sizeof(uint64_t)));
  return XG_OK;
}

template <typename E>
int launch_select(const ScanArgs& s, cudaStream_t stream) {
  const SelectArgs& a = s.a;
  const bool masked = a.masks.words || a.masks.slots;
  const unsigned grid = static_cast<unsigned>(a.groups) * a.beams * s.shares;
  static std::atomic<bool> allowed_scan[3][kDevices], allowed[kDevices];
  const auto scan = !masked ? scan_kernel<E, false, true> : a.renormalize ? scan_kernel<E, true, true> : scan_kernel<E, true, false>;
  if (int rc = allow_shared(reinterpret_cast<const void*>(scan), sizeof(ScanShared),
                            allowed_scan[!masked ? 0 : a.renormalize ? 1 : 2]))
    return rc;
  if (int rc = allow_shared(reinterpret_cast<const void*>(merge_kernel<E>), kPoolMax * 24, allowed)) return rc;
  cudaLaunchConfig_t config{};
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // a launch overlaps the end of what it waits for
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  config.stream = stream;
  config.gridDim = dim3(grid);
  config.blockDim = dim3(kScanThreads);
  config.dynamicSmemBytes = sizeof(ScanShared);
  XG_BEAM_CUDA(cudaLaunchKernelEx(&config, scan, s), "beam scan kernel");
  config.gridDim = dim3(static_cast<unsigned>(a.groups));
  config.blockDim = dim3(kMergeThreads);
  config.dynamicSmemBytes = static_cast<size_t>(s.pool) * 24;
  XG_BEAM_CUDA(cudaLaunchKernelEx(&config, merge_kernel<E>, s), "beam merge kernel");
  return XG_OK;
}

}  // namespace

int select(const SelectArgs& a, cudaStream_t stream) {
  if (int rc = check_sizes(a.groups, a.beams, a.vocab, a.dtype, a.candidates)) return rc;
  if (a.end_token < -1 || a.end_token >= a.vocab) return fail(XG_EINVAL, "end_token must be a token of the vocabulary, or -1");
  if (a.finished && a.end_token < 0) return fail(XG_EINVAL, "finished beams need end_token, the token they go on with");
  if (a.row_stride < a.vocab) return fail(XG_EINVAL, "logits need one contiguous row per beam");
  if (a.masks.words && a.masks.stride < (a.vocab + 31) / 32)
    return fail(XG_EINVAL, "the mask needs " + std::to_string((a.vocab + 31) / 32) + " words per row");
  if (a.groups == 0) return XG_OK;
  if (!a.logits || !a.scores || !a.out_scores || !a.out_beams || !a.out_tokens) return fail(XG_EINVAL, "null argument");
  if (reinterpret_cast<uintptr_t>(a.logits) % (a.dtype == XG_F32 ? 4 : 2))
    return fail(XG_EINVAL, "logits are not aligned to their element size");
  Plan p{};
  if (int rc = plan(a.groups, a.beams, a.vocab, a.dtype, a.candidates, &p)) return rc;
  if (!a.workspace || a.workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(a.workspace) % 16)
    return fail(XG_EINVAL, "the workspace needs " + std::to_string(p.bytes) + " bytes, 16-byte aligned");
  ScanArgs s{};
  s.a = a;
  const int64_t parts = static_cast<int64_t>(a.groups) * a.beams * p.shares;
  s.parts = reinterpret_cast<Part*>(a.workspace);
  s.keys = reinterpret_cast<uint64_t*>(a.workspace + parts * static_cast<int64_t>(sizeof(Part)));
  s.shares = p.shares;
  s.steps_per_share = p.steps_per_share;
  s.pool = p.pool;
  if (a.dtype == XG_F32) return launch_select<F32>(s, stream);
  if (a.dtype == XG_BF16) return launch_select<BF16>(s, stream);
  return launch_select<F16>(s, stream);
}

namespace {

struct Dim {
  int64_t size, stride;  // bytes
  bool position;
};

// One tensor's rows as at most two outer dimensions over a contiguous run: dimensions of one
// element drop out, neighbours that continue each other merge (but not across the position
// dimension's outer side, whose extent differs by group).
int describe(const XgRowTensor& t, bool has_lengths, MoveTensor* out, bool* empty) {
  const int32_t e = t.element_bytes;
  if (e != 1 && e != 2 && e != 4 && e != 8 && e != 16) return fail(XG_EINVAL, "elements must have 1, 2, 4, 8 or 16 bytes");
  if (t.dims < 0 || t.dims > 4) return fail(XG_EINVAL, "a row has at most 4 dimensions");
  if (t.position_dim < -1 || t.position_dim >= t.dims || (has_lengths && t.position_dim < 0))
    return fail(XG_EINVAL, "lengths need the tensors' position dimension");
  if (reinterpret_cast<uintptr_t>(t.data) % e) return fail(XG_EINVAL, "a tensor is not aligned to its element size");
  Dim d[4];
  int32_t n = 0;
  bool single = false;  // the position dimension has one place: a row moves if its length is not 0
  *empty = t.rows == 0;
  for (int32_t k = 0; k < t.dims; ++k) {
    if (t.size[k] < 0) return fail(XG_EINVAL, "negative size");
    if (t.size[k] == 0) *empty = true;
    if (t.stride[k] < 0) return fail(XG_EINVAL, "negative stride");
    const bool position = has_lengths && k == t.position_dim;
    if (t.size[k] == 1) {
      single = single || position;
      continue;
    }
    d[n++] = Dim{t.size[k], t.stride[k] * e, position};
  }
  if (*empty) return XG_OK;  // nothing to move, whatever the address: such tensors have none
  if (!t.data) return fail(XG_EINVAL, "null tensor");
  for (int32_t i = 1; i < n; ++i)  // the largest stride first: the order of a row's dimensions is free
    for (int32_t j = i; j > 0 && d[j].stride > d[j - 1].stride; --j) {
      const Dim x = d[j];
      d[j] = d[j - 1];
      d[j - 1] = x;
    }
  // no element twice: each stride clears what lies below it, and rows clear one another, or lie
  // inside the spaces between a row's own elements (a row dimension that is not outermost)
  int64_t below = e;
  bool row_placed = t.rows <= 1;
  for (int32_t i = n - 1; i >= 0; --i) {
    const int64_t row_stride = t.row_stride * e;
    if (!row_placed && row_stride < d[i].stride) {
      if (row_stride < below) return fail(XG_EINVAL, "a tensor's rows overlap");
      below += (t.rows - 1) * row_stride;
      row_placed = true;
    }
    if (d[i].stride < below) return fail(XG_EINVAL, "a tensor overlaps itself");
    below += (d[i].size - 1) * d[i].stride;
  }
  if (!row_placed && t.row_stride * e < below) return fail(XG_EINVAL, "a tensor's rows overlap");
  // the contiguous run, then the outer dimensions
  int64_t run = e, unit = 0;
  int32_t axis = single ? 4 : 0;
  while (n > 0 && d[n - 1].stride == run && axis != 3) {
    if (d[n - 1].position) {
      axis = 3;
      unit = run;
    }
    run *= d[n - 1].size;
    --n;
  }
  for (int32_t i = n - 1; i > 0; --i)
    if (!d[i].position && !d[i - 1].position && d[i - 1].stride == d[i].stride * d[i].size) {
      d[i - 1] = Dim{d[i - 1].size * d[i].size, d[i].stride, false};
      for (int32_t j = i; j + 1 < n; ++j) d[j] = d[j + 1];
      --n;
    }
  if (n > 2) return fail(XG_EINVAL, "a row's dimensions are strided in more than two places");
  MoveTensor m{};
  m.data = static_cast<char*>(t.data);
  m.row_bytes = t.row_stride * e;
  m.stride1 = n == 2 ? d[0].stride : 0;
  m.stride2 = n >= 1 ? d[n - 1].stride : 0;
  const int64_t size1 = n == 2 ? d[0].size : 1, size2 = n >= 1 ? d[n - 1].size : 1;
  if (n == 2 && d[0].position) axis = 1;
  if (n >= 1 && d[n - 1].position) axis = 2;
  // the widest access that everything is a multiple of
  uint64_t all = reinterpret_cast<uintptr_t>(t.data) | static_cast<uint64_t>(t.rows > 1 ? m.row_bytes : 0) |
                 static_cast<uint64_t>(run) | static_cast<uint64_t>(axis == 3 ? unit : 0) |
                 static_cast<uint64_t>(m.stride1) | static_cast<uint64_t>(m.stride2);
  int32_t log_bytes = 4;
  while (all & ((1u << log_bytes) - 1u)) --log_bytes;
  m.log_bytes = log_bytes;
  if (size1 > 0x7fffffff / size2 || (run >> log_bytes) > 0x7fffffff) return fail(XG_EINVAL, "a row is too large");
  m.size1 = static_cast<uint32_t>(size1);
  m.size2 = static_cast<uint32_t>(size2);
  m.size3 = static_cast<uint32_t>(run >> log_bytes);
  m.unit = static_cast<uint32_t>(unit >> log_bytes);
  m.axis = axis;
  *out = m;
  return XG_OK;
}

// A table of n words lies in a (described) tensor without gaps: the move would change it while it is read.
bool holds(const XgRowTensor& t, const int32_t* table, int64_t n) {
  if (!table || t.rows == 0) return false;
  int64_t elements = t.rows, extent = 1 + (t.rows - 1) * t.row_stride;
  for (int32_t k = 0; k < t.dims; ++k) {
    elements *= t.size[k];
    extent += (t.size[k] - 1) * t.stride[k];
  }
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.data), at = reinterpret_cast<uintptr_t>(table);
  return elements > 0 && elements == extent && at < begin + extent * t.element_bytes && begin < at + n * sizeof(int32_t);
}

int launch_moves(const MoveArgs& a, int64_t most_units, cudaStream_t stream) {
  int32_t sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  static std::atomic<bool> allowed[kDevices];
  if (int rc = allow_shared(reinterpret_cast<const void*>(move_kernel), kMaxBeams * kMoveThreads * 16, allowed)) return rc;
  // about one tile a CTA (with 0.6 parents a beam), so that groups with more to move do not hold
  // the others up; for huge tensors no more CTAs than keep every SM busy many times over
  const int64_t tile = static_cast<int64_t>(kMoveThreads) * a.slots * 10 / (a.beams * 6 + 4);
  const int64_t pairs = static_cast<int64_t>(a.groups) * a.count;
  int64_t shares = (most_units + tile - 1) / tile;
  const int64_t most = (static_cast<int64_t>(sms) * 128 + pairs - 1) / pairs;
  if (shares > most) shares = most;
  if (shares < 1) shares = 1;
  const dim3 grid(static_cast<unsigned>(shares), static_cast<unsigned>(a.groups), static_cast<unsigned>(a.count));
  move_kernel<<<grid, kMoveThreads, static_cast<size_t>(a.slots) * kMoveThreads * 16, stream>>>(a);
  XG_BEAM_CUDA(cudaGetLastError(), "beam reorder kernel");
  return XG_OK;
}

}  // namespace

int reorder(const XgRowTensor* tensors, int32_t count, const int32_t* parents, int32_t groups, int32_t beams,
            const int32_t* lengths, const int32_t* rows, cudaStream_t stream) {
  if (count < 0 || groups < 0 || beams < 1 || beams > kMaxBeams)
    return fail(XG_EINVAL, "a group holds 1 to " + std::to_string(kMaxBeams) + " beams, got " + std::to_string(beams));
  if (groups > 65535) return fail(XG_EINVAL, "at most 65535 groups");
  if (count == 0 || groups == 0) return XG_OK;
  if (!tensors || !parents) return fail(XG_EINVAL, "null argument");
  MoveArgs a;
  a.groups = groups;
  a.beams = beams;
  a.slots = beams > kMoveSlots ? beams : kMoveSlots;
  a.rows = tensors[0].rows;
  a.parents = parents;
  a.lengths = lengths;
  a.row_of = rows;
  const int64_t places = static_cast<int64_t>(groups) * beams;
  for (int32_t launches = 0; launches < 2; ++launches) {  // every descriptor is checked before the first launch
    if (launches)
      for (int32_t k = 0; k < count; ++k)
        if (holds(tensors[k], parents, places) || holds(tensors[k], lengths, groups) || holds(tensors[k], rows, places))
          return fail(XG_EINVAL, "parents, lengths and rows must not share memory with a tensor that is moved");
    a.count = 0;
    int64_t most_units = 0;
    for (int32_t k = 0; k < count; ++k) {
      if (tensors[k].rows != tensors[0].rows) return fail(XG_EINVAL, "the tensors of a call have the same number of rows");
      if (tensors[k].rows < (rows ? 0 : static_cast<int64_t>(groups) * beams) || tensors[k].rows > 0x7fffffff)
        return fail(XG_EINVAL, "the tensors need one row per beam");
      MoveTensor& m = a.tensors[a.count];
      bool empty = false;
      if (int rc = describe(tensors[k], lengths != nullptr, &m, &empty)) return rc;
      if (!empty) {
        const int64_t units = static_cast<int64_t>(m.size1) * m.size2 * m.size3;
        if (units > most_units) most_units = units;
        ++a.count;
      }
      if (a.count == kMoveTensors || (k + 1 == count && a.count > 0)) {
        if (launches)
          if (int rc = launch_moves(a, most_units, stream)) return rc;
        a.count = 0;
        most_units = 0;
      }
    }
  }
  return XG_OK;
}

}  // namespace beams
}  // namespace xg

using namespace xg::beams;

extern "C" XG_API int xg_beam_workspace(int32_t groups, int32_t beams, int32_t vocab, int32_t dtype, int32_t candidates,
                                        int64_t* bytes) {
  if (!bytes) return fail(XG_EINVAL, "null argument");
  if (int rc = check_sizes(groups, beams, vocab, dtype, candidates)) return rc;
  Plan p{};
  if (int rc = plan(groups, beams, vocab, dtype, candidates, &p)) return rc;
  *bytes = p.bytes;
  return XG_OK;
}

extern "C" XG_API int xg_beam_select(const void* logits, int32_t dtype, int32_t groups, int32_t beams, int32_t vocab,
                                     int64_t row_stride, const float* scores, const uint32_t* mask, int64_t mask_stride,
                                     const uint8_t* finished, int32_t candidates, int32_t end_token, int32_t renormalize,
                                     float* out_scores, int32_t* out_beams, int32_t* out_tokens, uint8_t* out_finished,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  SelectArgs a{};
  a.logits = static_cast<const char*>(logits);
  a.row_stride = row_stride;
  a.dtype = dtype;
  a.groups = groups;
  a.beams = beams;
  a.vocab = vocab;
  a.candidates = candidates;
  a.end_token = end_token;
  a.renormalize = renormalize != 0;
  a.scores = scores;
  a.finished = finished;
  a.masks.words = mask;
  a.masks.stride = mask_stride;
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  a.out_finished = out_finished;
  a.workspace = static_cast<char*>(workspace);
  a.workspace_bytes = workspace_bytes;
  return select(a, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" XG_API int xg_beam_reorder(const XgRowTensor* tensors, int32_t count, const int32_t* parents, int32_t groups,
                                      int32_t beams, const int32_t* lengths, const int32_t* rows, void* stream) {
  return reorder(tensors, count, parents, groups, beams, lengths, rows, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" XG_API int xg_beam_sequences(const int32_t* tokens, int64_t token_step, int64_t token_group,
                                        const int32_t* parents, int64_t parent_step, int64_t parent_group, int32_t steps,
                                        int32_t groups, int32_t beams, const int32_t* lengths, int32_t pad, int32_t* out,
                                        void* stream) {
  if (steps < 0 || groups < 0 || beams < 1 || beams > kMaxBeams)
    return fail(XG_EINVAL, "a group holds 1 to " + std::to_string(kMaxBeams) + " beams, got " + std::to_string(beams));
  if (groups > 0x7fffffff / 8) return fail(XG_EINVAL, "too many groups");
  if (steps == 0 || groups == 0) return XG_OK;
  if (!tokens || !parents || !out) return fail(XG_EINVAL, "null argument");
  TraceArgs a{};
  a.tokens = tokens;
  a.token_step = token_step;
  a.token_group = token_group;
  a.parents = parents;
  a.parent_step = parent_step;
  a.parent_group = parent_group;
  a.steps = steps;
  a.groups = groups;
  a.beams = beams;
  a.lengths = lengths;
  a.pad = pad;
  a.out = out;
  // a cluster of up to 8 CTAs a group, each with 64 steps or more of the trace
  a.cluster = 1;
  while (a.cluster < 8 && a.cluster * 64 < steps) a.cluster *= 2;
  a.window = (steps + a.cluster - 1) / a.cluster;
  const int32_t of_step = 6 * beams + 8;  // bytes, way_stride's rounding included
  if (a.window > kTraceBytes / of_step) a.window = kTraceBytes / of_step;
  a.way_stride = (((a.window + 3) / 4) | 1) * 4;  // an odd number of words: beams in different banks
  a.log_lanes = 0;
  while ((1 << a.log_lanes) < beams) ++a.log_lanes;
  // segments of about the square root of the window: the walks inside them and over them are alike
  a.segment = 8;
  while (a.segment * a.segment < a.window) a.segment *= 2;
  a.segments = (a.window + a.segment - 1) / a.segment;
  const int32_t bytes = a.window * (beams + 1) * 4 + a.window * beams + a.way_stride * beams + 2 * a.segments * beams +
                        (2 + a.cluster) * kMaxBeams;
  static std::atomic<bool> allowed[kDevices];
  if (int rc = allow_shared(reinterpret_cast<const void*>(trace_kernel), 2 * kTraceBytes, allowed)) return rc;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(groups) * a.cluster);
  config.blockDim = dim3(kTraceThreads);
  config.dynamicSmemBytes = static_cast<size_t>(bytes);
  config.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(a.cluster);
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  XG_BEAM_CUDA(cudaLaunchKernelEx(&config, trace_kernel, a), "beam sequences kernel");
  return XG_OK;
}
