// Beam search: selection over beams and vocabulary, reordering of per-beam state in place,
// and the back-trace of the written sequences (include/xgraph_b200.h has the definitions).
#include "beams.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <atomic>
#include <string>

extern "C" int xg_set_error(int code, const char* message);

namespace xg {
namespace beams {
namespace {

constexpr uint32_t kFull = 0xffffffffu;

// ---------------------------------------------------------------------------------------
// Selection, first kernel: every row's log-sum parts and its best tokens.
//
// A CTA streams a share of one row in tiles that stay in registers (kVecs 16-byte loads a
// thread, all in flight together), so each logit is read once: the tile's maximum and sum of
// exponentials, then its candidates, come from the same registers.

constexpr int32_t kScanThreads = 256;
constexpr int32_t kScanWarps = kScanThreads / 32;
constexpr int32_t kVecs = 8;          // 16-byte vectors a thread holds of a tile
constexpr int32_t kPushCap = 1024;    // candidates a tile may offer before the exact search takes over
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
__device__ __forceinline__ float exp2_fast(float x) {  // within 2 units of 2^-23 of 2^x
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

// How the three logit types sit in a 16-byte vector.
struct F32 {
  static constexpr int kPer = 4, kBytes = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  __device__ static float at(const uint4& v, int k) { return __uint_as_float((&v.x)[k]); }
  __device__ static float one(const char* p) { return *reinterpret_cast<const float*>(p); }
  __device__ static void put(uint4& v, int k, const char* p) { (&v.x)[k] = *reinterpret_cast<const uint32_t*>(p); }
  __device__ static float top(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
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
  __device__ static void put(uint4& v, int k, const char* p) {
    uint32_t& w = (&v.x)[k >> 1];
    const uint32_t b = *reinterpret_cast<const uint16_t*>(p);
    w = (k & 1) ? (w & 0x0000ffffu) | (b << 16) : (w & 0xffff0000u) | b;
  }
  __device__ static void keep(uint4& v, uint32_t bits) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t pair = bits >> (2 * k);
      const uint32_t m = ((pair & 1u) ? 0x0000ffffu : 0u) | ((pair & 2u) ? 0xffff0000u : 0u);
      (&v.x)[k] = ((&v.x)[k] & m) | (kNegInf & ~m);
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
  __device__ static float top(const uint4& v) {
    const auto h = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h(v.x), h(v.y)), __hmax2_nan(h(v.z), h(v.w)));
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
  __device__ static float top(const uint4& v) {
    const auto h = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
    const __half2 m = __hmax2_nan(__hmax2_nan(h(v.x), h(v.y)), __hmax2_nan(h(v.z), h(v.w)));
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

// What the scan leaves for the merge: per (row, share) the log-sum parts, and its best keys,
// best first (rising(logit) << 32 | ~token; 0: none).
struct Part {
  double sum;  // of exp(x - top)
  float top;
  int32_t pad;
};

struct ScanArgs {
  SelectArgs a;
  Part* parts;      // [rows][shares]
  uint64_t* keys;   // [rows][shares][candidates]
  int32_t shares, tiles_per_share;
  int32_t pool;     // beams * shares * candidates
};

__device__ __forceinline__ uint64_t make_key(uint32_t order, int32_t token) {
  return (static_cast<uint64_t>(order) << 32) | static_cast<uint32_t>(~token);
}

// Row r takes part: its score is finite and the beam has not ended.
__device__ __forceinline__ bool row_scans(const SelectArgs& a, int32_t row) {
  const bool ended = a.finished && a.finished[row];
  return isfinite(a.scores[row]) && !ended;
}

struct ScanShared {
  uint64_t pushed[kPushCap];
  uint64_t best[2][kMaxCandidates];
  uint32_t group_top[kMaxCandidates];  // the maxima of the groups a tile's threads form
  double warp_sum[kScanWarps];
  float warp_top[kScanWarps];
  int32_t counts[2][kScanWarps];
  int32_t count;
};

__device__ __forceinline__ int32_t block_total(int32_t mine, int32_t (&counts)[kScanWarps]) {
  const int32_t of_warp = __reduce_add_sync(kFull, mine);
  if ((threadIdx.x & 31) == 0) counts[threadIdx.x >> 5] = of_warp;
  __syncthreads();
  int32_t total = 0;
#pragma unroll
  for (int32_t w = 0; w < kScanWarps; ++w) total += counts[w];
  return total;
}

template <typename E, bool MASKED, bool RENORMALIZE>
__global__ void __launch_bounds__(kScanThreads, 3) scan_kernel(const __grid_constant__ ScanArgs s) {
  __shared__ ScanShared sh;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the merge waits for this grid's end
  constexpr int32_t kPer = E::kPer;
  constexpr int32_t kTileVecs = kScanThreads * kVecs;
  const SelectArgs& a = s.a;
  const int32_t row = blockIdx.x / s.shares, share = blockIdx.x - row * s.shares;
  if (!row_scans(a, row)) return;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t wanted = a.candidates, vocab = a.vocab;
  const char* logits = a.logits + static_cast<int64_t>(row) * a.row_stride * E::kBytes;
  // vectors start at 16-byte boundaries, so the first may begin before the row
  const int32_t head = static_cast<int32_t>(reinterpret_cast<uintptr_t>(logits) & 15u) / E::kBytes;
  const int32_t vecs = (vocab + head + kPer - 1) / kPer;
  const RowMask mask = MASKED ? row_mask(a.masks, row) : RowMask{nullptr, nullptr};
  // candidates need a bound that at least `wanted` of a tile's tokens reach: the least of the
  // maxima of `groups` groups of threads, with groups >= wanted
  int32_t groups = kScanWarps;
  while (groups < wanted) groups <<= 1;
  const int32_t group_lanes = kScanThreads / groups;

  double sum = 0.0;                       // of this warp's tokens so far, relative to `top`
  float top = -CUDART_INF_F;
  int32_t held = 0, which = 0;            // sh.best[which] holds the best so far
  uint32_t bar = kRisingLowest;           // tokens below it cannot be among the best

  const int32_t tile_end = min((share + 1) * s.tiles_per_share, (vecs + kTileVecs - 1) / kTileVecs);
  for (int32_t tile = share * s.tiles_per_share; tile < tile_end; ++tile) {
    const int32_t v0 = tile * kTileVecs + tid;
    uint4 v[kVecs];
    uint32_t bits[kVecs];
#pragma unroll
    for (int32_t j = 0; j < kVecs; ++j) {
      const int32_t t0 = (v0 + j * kScanThreads) * kPer - head;
      bits[j] = t0 >= vocab ? 0u : MASKED ? mask.bits(t0, kPer, vocab) : RowMask{nullptr, nullptr}.bits(t0, kPer, vocab);
    }
#pragma unroll
    for (int32_t j = 0; j < kVecs; ++j) {
      const int32_t t0 = (v0 + j * kScanThreads) * kPer - head;
      v[j] = make_uint4(E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf);
      if (t0 >= vocab || (RENORMALIZE && bits[j] == 0u)) continue;
      const char* at = logits + static_cast<int64_t>(t0) * E::kBytes;
      if (t0 >= 0 && t0 + kPer <= vocab) {
        v[j] = __ldcs(reinterpret_cast<const uint4*>(at));
      } else {
#pragma unroll
        for (int32_t k = 0; k < kPer; ++k)
          if (t0 + k >= 0 && t0 + k < vocab) E::put(v[j], k, at + k * E::kBytes);
      }
    }
    if (MASKED && RENORMALIZE) {
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j)
        if (bits[j] != (1u << kPer) - 1u) E::keep(v[j], bits[j]);
    }
    // the tile's maximum and sum, per warp: exp(x - m) as 2^(x log2 e - a) with a the float
    // nearest m log2 e, so that the shared part of every exponent is exact
    float most = E::top(v[0]);
#pragma unroll
    for (int32_t j = 1; j < kVecs; ++j) most = max_nan(most, E::top(v[j]));
    float shown = most;
#pragma unroll
    for (int32_t d = 16; d > 0; d >>= 1) most = max_nan(most, __shfl_xor_sync(kFull, most, d));
    if (most != -CUDART_INF_F) {  // uniform in the warp
      double part;
      if (fabsf(most) < 65536.0f) {
        const float anchor = __fmul_rn(most, kLog2eHi);
        const uint64_t hi = pack2(kLog2eHi, kLog2eHi), lo = pack2(kLog2eLo, kLog2eLo), back = pack2(-anchor, -anchor);
        uint64_t acc[2] = {0, 0};
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j) {
#pragma unroll
          for (int32_t k = 0; k < kPer; k += 2) {
            const uint64_t x = pack2(E::at(v[j], k), E::at(v[j], k + 1));
            const uint64_t y = fma2(x, lo, fma2(x, hi, back));
            acc[(k >> 1) & 1] = add2(acc[(k >> 1) & 1], pack2(exp2_fast(low(y)), exp2_fast(high(y))));
          }
        }
        const uint64_t all = add2(acc[0], acc[1]);
        part = static_cast<double>(low(all)) + static_cast<double>(high(all));
#pragma unroll
        for (int32_t d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(kFull, part, d);
        part *= exp(static_cast<double>(anchor) * 0.69314718055994530942 - static_cast<double>(most));
      } else {  // far from 0 (or not finite) the difference comes first
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j) {
#pragma unroll
          for (int32_t k = 0; k < kPer; ++k) {
            const float d = E::at(v[j], k) - most;
            acc[k & 3] += exp2_fast(fmaf(d, kLog2eHi, d * kLog2eLo));
          }
        }
        part = static_cast<double>(acc[0] + acc[1]) + static_cast<double>(acc[2] + acc[3]);
#pragma unroll
        for (int32_t d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(kFull, part, d);
      }
      if (top == -CUDART_INF_F) {
        sum = part;
        top = most;
      } else {
        const float higher = max_nan(top, most);
        sum = sum * exp(static_cast<double>(top) - static_cast<double>(higher)) +
              part * exp(static_cast<double>(most) - static_cast<double>(higher));
        top = higher;
      }
    }
    if (MASKED && !RENORMALIZE) {
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j)
        if (bits[j] != (1u << kPer) - 1u) E::keep(v[j], bits[j]);
      shown = E::top(v[0]);
#pragma unroll
      for (int32_t j = 1; j < kVecs; ++j) shown = max_nan(shown, E::top(v[j]));
    }
    // the bound, then every token that reaches it
    uint32_t group = rising(shown + 0.0f);
    for (int32_t d = 1; d < group_lanes; d <<= 1) group = max(group, __shfl_xor_sync(kFull, group, d));
    if ((lane & (group_lanes - 1)) == 0) sh.group_top[tid / group_lanes] = group;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    uint32_t bound = kFull;
    for (int32_t g = lane; g < groups; g += 32) bound = min(bound, sh.group_top[g]);
    bound = max(__reduce_min_sync(kFull, bound), bar);
    const float reach = from_rising(bound);
    if (shown >= reach) {
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j) {
        if (!(E::top(v[j]) >= reach)) continue;
        const int32_t t0 = (v0 + j * kScanThreads) * kPer - head;
#pragma unroll
        for (int32_t k = 0; k < kPer; ++k) {
          const float x = E::at(v[j], k) + 0.0f;
          if (x >= reach) {
            const int32_t n = atomicAdd(&sh.count, 1);
            if (n < kPushCap) sh.pushed[n] = make_key(rising(x), t0 + k);
          }
        }
      }
    }
    __syncthreads();
    int32_t pushed = sh.count;
    if (pushed > kPushCap) {
      // too many reach it (ties, or few allowed groups): the exact `wanted`-th best order
      // number by bisection, then the token bound among its equals
      uint32_t edge = 0;
      int32_t turn = 0;
      for (int32_t bit = 31; bit >= 0; --bit, turn ^= 1) {
        const uint32_t trial = edge | (1u << bit);
        int32_t mine = 0;
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j)
#pragma unroll
          for (int32_t k = 0; k < kPer; ++k) mine += rising(E::at(v[j], k) + 0.0f) >= trial;
        if (block_total(mine, sh.counts[turn]) >= wanted) edge = trial;
      }
      int32_t above = 0;
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j)
#pragma unroll
        for (int32_t k = 0; k < kPer; ++k) above += rising(E::at(v[j], k) + 0.0f) > edge;
      above = block_total(above, sh.counts[turn]);
      turn ^= 1;
      int32_t lowest = -1;  // equals up to lowest + 1 are taken
      for (int32_t bit = 20; bit >= 0; --bit, turn ^= 1) {
        const int32_t trial = lowest + (1 << bit);
        int32_t mine = 0;
#pragma unroll
        for (int32_t j = 0; j < kVecs; ++j)
#pragma unroll
          for (int32_t k = 0; k < kPer; ++k)
            mine += rising(E::at(v[j], k) + 0.0f) == edge && (v0 + j * kScanThreads) * kPer - head + k <= trial;
        if (block_total(mine, sh.counts[turn]) < wanted - above) lowest = trial;
      }
      if (tid == 0) sh.count = 0;
      __syncthreads();
#pragma unroll
      for (int32_t j = 0; j < kVecs; ++j) {
        const int32_t t0 = (v0 + j * kScanThreads) * kPer - head;
#pragma unroll
        for (int32_t k = 0; k < kPer; ++k) {
          const uint32_t o = rising(E::at(v[j], k) + 0.0f);
          if (o > edge || (o == edge && t0 + k <= lowest + 1)) {
            const int32_t n = atomicAdd(&sh.count, 1);
            if (n < kPushCap) sh.pushed[n] = make_key(o, t0 + k);
          }
        }
      }
      __syncthreads();
      pushed = min(sh.count, kPushCap);
    }
    // the best of those held and those pushed, in order, by counting the greater ones
    const int32_t n = held + pushed;
    const uint64_t* old = sh.best[which];
    uint64_t* fresh = sh.best[which ^ 1];
    for (int32_t i = tid; i < n; i += kScanThreads) {
      const uint64_t mine = i < held ? old[i] : sh.pushed[i - held];
      int32_t rank = 0;
      for (int32_t j = 0; j < held; ++j) rank += old[j] > mine;
      for (int32_t j = 0; j < pushed; ++j) rank += sh.pushed[j] > mine;
      if (rank < wanted) fresh[rank] = mine;
    }
    __syncthreads();
    which ^= 1;
    held = min(n, wanted);
    // a later token equal to the last of a full list comes after it
    if (held == wanted) bar = max(bar, static_cast<uint32_t>(fresh[wanted - 1] >> 32) + 1u);
  }
  if (lane == 0) {
    sh.warp_top[warp] = top;
    sh.warp_sum[warp] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    const float t = lane < kScanWarps ? sh.warp_top[lane] : -CUDART_INF_F;
    float most = t;
#pragma unroll
    for (int32_t d = 16; d > 0; d >>= 1) most = max_nan(most, __shfl_xor_sync(kFull, most, d));
    double part = 0.0;
    if (lane < kScanWarps && t != -CUDART_INF_F)
      part = sh.warp_sum[lane] * exp(static_cast<double>(t) - static_cast<double>(most));
#pragma unroll
    for (int32_t d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(kFull, part, d);
    if (lane == 0) s.parts[blockIdx.x] = Part{part, most, 0};
  }
  uint64_t* out = s.keys + static_cast<int64_t>(blockIdx.x) * wanted;
  for (int32_t i = tid; i < wanted; i += kScanThreads) out[i] = i < held ? sh.best[which][i] : 0u;
}

// ---------------------------------------------------------------------------------------
// Selection, second kernel: one CTA per group scores the rows' candidates in 64 bits and
// orders the best.

constexpr int32_t kMergeThreads = 512;
constexpr int32_t kMergeWarps = kMergeThreads / 32;
constexpr int32_t kSamples = 1024;
// Two beams' candidates nearer than this are ordered by log-sums taken again in 64 bits.
constexpr double kNear = 1e-6;

struct MergeShared {
  double sample[kSamples];
  double log_sum[kMaxBeams];
  double score[kMaxBeams];
  float top[kMaxBeams];
  int32_t state[kMaxBeams];   // 0 offers nothing, 1 candidates, 2 ended, 3 candidates, 64-bit sum
  int32_t again[kMaxBeams];
  int32_t order[kMaxCandidates + 1];
  double warp_sum[kMergeWarps];
  double bound;
  int32_t count, near;
};

// Sum over N_r of exp(x - top) in 64 bits, by the whole CTA.
template <typename E>
__device__ double row_sum(const SelectArgs& a, int32_t row, float top, double (&scratch)[kMergeWarps]) {
  const char* logits = a.logits + static_cast<int64_t>(row) * a.row_stride * E::kBytes;
  const RowMask mask = a.renormalize ? row_mask(a.masks, row) : RowMask{nullptr, nullptr};
  double sum = 0.0;
  for (int32_t t = threadIdx.x; t < a.vocab; t += kMergeThreads) {
    if (!mask.all() && !((mask.word(t >> 5) >> (t & 31)) & 1u)) continue;
    sum += exp(static_cast<double>(E::one(logits + static_cast<int64_t>(t) * E::kBytes)) - static_cast<double>(top));
  }
#pragma unroll
  for (int32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int32_t w = 0; w < kMergeWarps; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

template <typename E>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const __grid_constant__ ScanArgs s) {
  extern __shared__ __align__(16) char dynamic[];
  __shared__ MergeShared sh;
  const SelectArgs& a = s.a;
  const int32_t pool = s.pool, beams = a.beams, shares = s.shares, wanted = a.candidates;
  double* value = reinterpret_cast<double*>(dynamic);            // [pool]; -inf: none
  uint32_t* code = reinterpret_cast<uint32_t*>(value + pool);    // [pool] beam << 20 | token
  int32_t* kept = reinterpret_cast<int32_t*>(code + pool);       // [pool] places above the bound
  const int32_t group = blockIdx.x, row0 = group * beams;
  const int32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the scan is complete

  for (int32_t b = warp; b < beams; b += kMergeWarps) {
    const int32_t row = row0 + b;
    const float score = a.scores[row];
    int32_t state = 0;
    float top = -CUDART_INF_F;
    double sum = 0.0;
    if (isfinite(score)) {
      if (a.finished && a.finished[row]) {
        state = 2;
      } else {
        for (int32_t c = lane; c < shares; c += 32) top = max_nan(top, s.parts[row * shares + c].top);
#pragma unroll
        for (int32_t d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(kFull, top, d));
        for (int32_t c = lane; c < shares; c += 32) {
          const Part p = s.parts[row * shares + c];
          if (p.top != -CUDART_INF_F) sum += p.sum * exp(static_cast<double>(p.top) - static_cast<double>(top));
        }
#pragma unroll
        for (int32_t d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
        state = isfinite(sum) && sum > 0.0 ? 1 : 0;
      }
    }
    if (lane == 0) {
      sh.score[b] = score;
      sh.state[b] = state;
      sh.top[b] = top;
      sh.log_sum[b] = state == 1 ? log(sum) : 0.0;
    }
  }
  const int32_t lists = beams * shares;
  for (;;) {
    __syncthreads();
    for (int32_t i = tid; i < pool; i += kMergeThreads) {
      const int32_t list = i / wanted, place = i - list * wanted;
      const int32_t b = list / shares, state = sh.state[b];
      double v = -CUDART_INF;
      int32_t token = 0;
      if (state == 2) {
        if (place == 0 && list - b * shares == 0 && a.end_token >= 0) {
          v = sh.score[b];
          token = a.end_token;
        }
      } else if (state) {
        const uint64_t key = s.keys[static_cast<int64_t>(row0) * shares * wanted + i];
        if (key) {
          token = static_cast<int32_t>(~static_cast<uint32_t>(key));
          const float x = from_rising(static_cast<uint32_t>(key >> 32));
          v = sh.score[b] + ((static_cast<double>(x) - static_cast<double>(sh.top[b])) - sh.log_sum[b]);
          if (!isfinite(__double2float_rn(v))) v = -CUDART_INF;
        }
      }
      value[i] = v;
      code[i] = (static_cast<uint32_t>(b) << 20) | static_cast<uint32_t>(token);
    }
    if (tid == 0) sh.count = sh.near = 0;
    __syncthreads();
    // a bound that `wanted` candidates reach: the wanted-th best of a sample of distinct ones,
    // the lists' first places (their maxima over 4 * wanted sets of lists, if there are more)
    const int32_t target = 4 * wanted;
    int32_t samples;
    if (lists >= target) {
      samples = target;
      for (int32_t i = tid; i < samples; i += kMergeThreads) {
        double most = -CUDART_INF;
        for (int32_t l = i; l < lists; l += target) most = fmax(most, value[l * wanted]);
        sh.sample[i] = most;
      }
    } else {
      const int32_t places = min((target + lists - 1) / lists, wanted);
      samples = lists * places;  // at most target + lists <= 8 * wanted <= kSamples
      for (int32_t i = tid; i < samples; i += kMergeThreads) {
        const int32_t l = i / places;
        sh.sample[i] = value[l * wanted + (i - l * places)];
      }
    }
    if (tid == 0) sh.bound = -CUDART_INF;
    __syncthreads();
    for (int32_t i = tid; i < samples; i += kMergeThreads) {
      const double mine = sh.sample[i];
      int32_t rank = 0;
      for (int32_t j = 0; j < samples; ++j) rank += sh.sample[j] > mine || (sh.sample[j] == mine && j < i);
      if (rank == wanted - 1) sh.bound = mine;
    }
    __syncthreads();
    const double bound = sh.bound - 2.0 * kNear;
    for (int32_t i = tid; i < pool; i += kMergeThreads)
      if (value[i] > -CUDART_INF && value[i] >= bound) kept[atomicAdd(&sh.count, 1)] = i;
    __syncthreads();
    const int32_t n = sh.count;
    for (int32_t i = tid; i < n; i += kMergeThreads) {
      const int32_t at = kept[i];
      const double mine = value[at];
      const uint32_t own = code[at];
      int32_t rank = 0;
      for (int32_t j = 0; j < n; ++j) {
        const double other = value[kept[j]];
        rank += other > mine || (other == mine && code[kept[j]] < own);
      }
      if (rank <= wanted) sh.order[rank] = at;
    }
    for (int32_t b = tid; b < beams; b += kMergeThreads) sh.again[b] = 0;
    __syncthreads();
    // neighbours of different beams whose order the 32-bit sums cannot tell
    const int32_t listed = min(n, wanted + 1);
    for (int32_t i = tid; i + 1 < listed; i += kMergeThreads) {
      const int32_t p = sh.order[i], q = sh.order[i + 1];
      const int32_t bp = code[p] >> 20, bq = code[q] >> 20;
      if (bp != bq && value[p] - value[q] <= kNear) {
        if (sh.state[bp] == 1) sh.again[bp] = sh.near = 1;
        if (sh.state[bq] == 1) sh.again[bq] = sh.near = 1;
      }
    }
    __syncthreads();
    if (!sh.near) break;
    for (int32_t b = 0; b < beams; ++b) {  // at most once for each beam
      if (!sh.again[b]) continue;
      const double sum = row_sum<E>(a, row0 + b, sh.top[b], sh.warp_sum);
      if (tid == 0) {
        sh.log_sum[b] = log(sum);
        sh.state[b] = 3;
      }
    }
  }
  for (int32_t i = tid; i < wanted; i += kMergeThreads) {
    const int64_t to = static_cast<int64_t>(group) * wanted + i;
    float score = -CUDART_INF_F;
    int32_t beam = -1, token = -1;
    bool ended = false;
    if (i < sh.count) {
      const int32_t at = sh.order[i];
      score = __double2float_rn(value[at]);
      beam = static_cast<int32_t>(code[at] >> 20);
      token = static_cast<int32_t>(code[at] & 0xfffffu);
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
// A thread owns one unit (up to 16 bytes) of every row of a group: it loads the unit from
// each moved row's parent, then stores them, so the move is in place without a copy of the
// rows, whatever cycles the parents form, and each byte that stays is not touched.

constexpr int32_t kMoveThreads = 256;
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
  int32_t count, groups, beams;
  int64_t rows;
  const int32_t* parents;
  const int32_t* lengths;
  const int32_t* row_of;
};

template <int32_t MOST, typename V>
__device__ __forceinline__ void move_unit(const MoveTensor& t, int64_t offset, int32_t moved, const int32_t* from,
                                          const int32_t* to) {
  V held[MOST];
  char* at = t.data + offset;
#pragma unroll
  for (int32_t i = 0; i < MOST; ++i)
    if (i < moved) held[i] = *reinterpret_cast<const V*>(at + from[i] * t.row_bytes);
#pragma unroll
  for (int32_t i = 0; i < MOST; ++i)
    if (i < moved) *reinterpret_cast<V*>(at + to[i] * t.row_bytes) = held[i];
}

template <int32_t MOST>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveArgs a) {
  __shared__ int32_t from[kMaxBeams], to[kMaxBeams];
  __shared__ int32_t moves;
  const int32_t group = blockIdx.y;
  if (threadIdx.x < 32) {
    int32_t n = 0;
    for (int32_t b0 = 0; b0 < a.beams; b0 += 32) {
      const int32_t b = b0 + static_cast<int32_t>(threadIdx.x);
      int32_t source = -1, target = -1;
      if (b < a.beams) {
        const int32_t parent = a.parents[group * a.beams + b];
        if (parent >= 0 && parent < a.beams && parent != b) {
          source = group * a.beams + parent;
          target = group * a.beams + b;
          if (a.row_of) {
            source = a.row_of[source];
            target = a.row_of[target];
          }
        }
      }
      const bool valid = source >= 0 && source < a.rows && target >= 0 && target < a.rows && source != target;
      const uint32_t who = __ballot_sync(kFull, valid);
      if (valid) {
        const int32_t at = n + __popc(who & ((1u << threadIdx.x) - 1u));
        from[at] = source;
        to[at] = target;
      }
      n += __popc(who);
    }
    if (threadIdx.x == 0) moves = n;
  }
  __syncthreads();
  const int32_t moved = moves;
  if (moved == 0) return;
  const int32_t length = a.lengths ? max(a.lengths[group], 0) : 0x7fffffff;
  uint64_t next = blockIdx.x, first = 0;
  for (int32_t k = 0; k < a.count; ++k) {
    const MoveTensor& t = a.tensors[k];
    const uint32_t size1 = t.axis == 1 ? min(t.size1, static_cast<uint32_t>(length)) : t.size1;
    const uint32_t size2 = t.axis == 2 ? min(t.size2, static_cast<uint32_t>(length)) : t.size2;
    const uint32_t size3 =
        t.axis == 3 ? static_cast<uint32_t>(min(static_cast<uint64_t>(t.size3), static_cast<uint64_t>(t.unit) * length))
                    : t.size3;
    const uint64_t units = t.axis == 4 && length == 0 ? 0 : static_cast<uint64_t>(size1) * size2 * size3;
    const uint64_t tiles = (units + kMoveThreads - 1) / kMoveThreads;
    for (; next < first + tiles; next += gridDim.x) {
      const uint64_t unit = (next - first) * kMoveThreads + threadIdx.x;
      if (unit >= units) continue;
      int64_t offset;
      if (size3 == units) {
        offset = static_cast<int64_t>(unit) << t.log_bytes;
      } else {
        const uint64_t outer = unit / size3;
        const uint32_t i1 = static_cast<uint32_t>(outer / size2), i2 = static_cast<uint32_t>(outer - static_cast<uint64_t>(i1) * size2);
        offset = i1 * t.stride1 + i2 * t.stride2 + (static_cast<int64_t>(unit - outer * size3) << t.log_bytes);
      }
      switch (t.log_bytes) {
        case 4:
          if constexpr (MOST <= 32) move_unit<MOST, uint4>(t, offset, moved, from, to);
          break;
        case 3: move_unit<MOST, uint2>(t, offset, moved, from, to); break;
        case 2: move_unit<MOST, uint32_t>(t, offset, moved, from, to); break;
        case 1: move_unit<MOST, uint16_t>(t, offset, moved, from, to); break;
        default: move_unit<MOST, uint8_t>(t, offset, moved, from, to); break;
      }
    }
    first += tiles;
  }
}

// ---------------------------------------------------------------------------------------
// The back-trace.

constexpr int32_t kTraceThreads = 512;
constexpr int32_t kTraceBytes = 96 * 1024;  // shared memory for a window's parents
constexpr uint8_t kNoBeam = 0xff;

struct TraceArgs {
  const int32_t* tokens;
  int64_t token_step, token_group;
  const int32_t* parents;
  int64_t parent_step, parent_group;
  int32_t steps, groups, beams;
  const int32_t* lengths;
  int32_t pad, window, segment;
  int32_t* out;
};

// One CTA per group, windows of steps from the last to the first.  A window's parent maps sit
// in shared memory as bytes; its segments are walked in parallel twice: once from every
// beam, which gives each segment's map, and, after the maps are chained, once more along the
// beams that each last place came through, which leaves every step's beam in shared memory
// for the tokens' gather.
__global__ void __launch_bounds__(kTraceThreads) trace_kernel(const __grid_constant__ TraceArgs a) {
  extern __shared__ __align__(16) uint8_t maps[];  // [window][beams], then [window][beams] ways, then segments' maps
  const int32_t group = blockIdx.x, beams = a.beams, tid = threadIdx.x;
  const int32_t length = a.lengths ? min(max(a.lengths[group], 0), a.steps) : a.steps;
  uint8_t* way = maps + a.window * beams;
  const int32_t segments_most = (a.window + a.segment - 1) / a.segment;
  uint8_t* through = way + a.window * beams;              // [segments][beams]: from the segment's end to before it
  uint8_t* enter = through + segments_most * beams;       // [segments][beams]: the beam at the segment's end, per last place
  uint8_t* carry = enter + segments_most * beams;         // [beams]: the beam at the window's end, per last place
  int32_t* out = a.out + static_cast<int64_t>(group) * beams * a.steps;
  for (int64_t i = tid; i < static_cast<int64_t>(beams) * (a.steps - length); i += kTraceThreads) {
    const int32_t k = static_cast<int32_t>(i / (a.steps - length));
    out[static_cast<int64_t>(k) * a.steps + length + (i - static_cast<int64_t>(k) * (a.steps - length))] = a.pad;
  }
  for (int32_t k = tid; k < beams; k += kTraceThreads) carry[k] = static_cast<uint8_t>(k);
  for (int32_t end = length; end > 0; end -= a.window) {
    const int32_t begin = max(0, end - a.window), count = end - begin;
    const int32_t segments = (count + a.segment - 1) / a.segment;
    __syncthreads();
    for (int32_t i = tid; i < count * beams; i += kTraceThreads) {
      const int32_t t = i / beams, k = i - t * beams;
      const int32_t p = a.parents[(begin + t) * a.parent_step + group * a.parent_group + k];
      maps[i] = p >= 0 && p < beams ? static_cast<uint8_t>(p) : kNoBeam;
    }
    __syncthreads();
    for (int32_t i = tid; i < segments * beams; i += kTraceThreads) {
      const int32_t s = i / beams;
      const int32_t t0 = s * a.segment, t1 = min(t0 + a.segment, count);
      uint8_t at = static_cast<uint8_t>(i - s * beams);
      for (int32_t t = t1 - 1; t >= t0 && at != kNoBeam; --t) at = maps[t * beams + at];
      through[i] = at;
    }
    __syncthreads();
    if (tid < beams) {
      uint8_t at = carry[tid];
      for (int32_t s = segments - 1; s >= 0; --s) {
        enter[s * beams + tid] = at;
        if (at != kNoBeam) at = through[s * beams + at];
      }
      carry[tid] = at;
    }
    __syncthreads();
    for (int32_t i = tid; i < segments * beams; i += kTraceThreads) {
      const int32_t s = i / beams, k = i - s * beams;
      const int32_t t0 = s * a.segment, t1 = min(t0 + a.segment, count);
      uint8_t at = enter[i];
      for (int32_t t = t1 - 1; t >= t0; --t) {
        way[t * beams + k] = at;
        if (at != kNoBeam) at = maps[t * beams + at];
      }
    }
    __syncthreads();
    for (int32_t i = tid; i < count * beams; i += kTraceThreads) {
      const int32_t k = i / count, t = i - k * count;
      const uint8_t at = way[t * beams + k];
      out[static_cast<int64_t>(k) * a.steps + begin + t] =
          at == kNoBeam ? a.pad : a.tokens[(begin + t) * a.token_step + group * a.token_group + at];
    }
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
  int32_t shares, tiles_per_share, pool;
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
  // a misaligned row's vectors may start a vector early
  const int32_t tiles = (vocab + 2 * per - 1) / per / (kScanThreads * kVecs) + 1;
  const int64_t rows = static_cast<int64_t>(groups) * beams;
  int64_t shares = rows > 0 ? (static_cast<int64_t>(sms) * 8 + rows - 1) / rows : 1;
  if (shares > kPoolMax / (beams * candidates)) shares = kPoolMax / (beams * candidates);
  if (shares > tiles) shares = tiles;
  if (shares < 1) shares = 1;
  out->tiles_per_share = static_cast<int32_t>((tiles + shares - 1) / shares);
  out->shares = (tiles + out->tiles_per_share - 1) / out->tiles_per_share;
  out->pool = beams * out->shares * candidates;
  out->bytes = rows * out->shares * (static_cast<int64_t>(sizeof(Part)) + candidates * static_cast<int64_t>(sizeof(uint64_t)));
  return XG_OK;
}

template <typename E>
int launch_select(const ScanArgs& s, cudaStream_t stream) {
  const SelectArgs& a = s.a;
  const bool masked = a.masks.words || a.masks.slots;
  const unsigned grid = static_cast<unsigned>(a.groups) * a.beams * s.shares;
  if (!masked)
    scan_kernel<E, false, true><<<grid, kScanThreads, 0, stream>>>(s);
  else if (a.renormalize)
    scan_kernel<E, true, true><<<grid, kScanThreads, 0, stream>>>(s);
  else
    scan_kernel<E, true, false><<<grid, kScanThreads, 0, stream>>>(s);
  XG_BEAM_CUDA(cudaGetLastError(), "beam scan kernel");
  static std::atomic<bool> allowed[kDevices];
  if (int rc = allow_shared(reinterpret_cast<const void*>(merge_kernel<E>), kPoolMax * 16, allowed)) return rc;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.groups));
  config.blockDim = dim3(kMergeThreads);
  config.dynamicSmemBytes = static_cast<size_t>(s.pool) * 16;
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its launch overlaps the scan's end
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
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
  s.tiles_per_share = p.tiles_per_share;
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
int describe(const XgRowTensor& t, bool has_lengths, int32_t beams, MoveTensor* out, bool* empty) {
  const int32_t e = t.element_bytes;
  if (!t.data) return fail(XG_EINVAL, "null tensor");
  if (e != 1 && e != 2 && e != 4 && e != 8 && e != 16) return fail(XG_EINVAL, "elements must have 1, 2, 4, 8 or 16 bytes");
  if (t.dims < 0 || t.dims > 4) return fail(XG_EINVAL, "a row has at most 4 dimensions");
  if (t.position_dim < -1 || t.position_dim >= t.dims || (has_lengths && t.position_dim < 0))
    return fail(XG_EINVAL, "lengths need the tensors' position dimension");
  if (reinterpret_cast<uintptr_t>(t.data) % e) return fail(XG_EINVAL, "a tensor is not aligned to its element size");
  Dim d[4];
  int32_t n = 0;
  bool single = false;  // the position dimension has one place: a row moves if its length is not 0
  *empty = false;
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
  if (*empty) return XG_OK;
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
  // the widest access that everything is a multiple of (16 bytes for 33 beams and more would
  // take more registers than a thread has)
  uint64_t all = reinterpret_cast<uintptr_t>(t.data) | static_cast<uint64_t>(t.rows > 1 ? m.row_bytes : 0) |
                 static_cast<uint64_t>(run) | static_cast<uint64_t>(axis == 3 ? unit : 0) |
                 static_cast<uint64_t>(m.stride1) | static_cast<uint64_t>(m.stride2);
  int32_t log_bytes = beams > 32 ? 3 : 4;
  while (all & ((1u << log_bytes) - 1u)) --log_bytes;
  m.log_bytes = log_bytes;
  if (size1 > 0x7fffffff || size2 > 0x7fffffff || (run >> log_bytes) > 0x7fffffff || (unit >> log_bytes) > 0x7fffffff)
    return fail(XG_EINVAL, "a row is too large");
  m.size1 = static_cast<uint32_t>(size1);
  m.size2 = static_cast<uint32_t>(size2);
  m.size3 = static_cast<uint32_t>(run >> log_bytes);
  m.unit = static_cast<uint32_t>(unit >> log_bytes);
  m.axis = axis;
  *out = m;
  return XG_OK;
}

int launch_moves(const MoveArgs& a, int64_t units, cudaStream_t stream) {
  int32_t sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int64_t tiles = (units + kMoveThreads - 1) / kMoveThreads;
  int64_t shares = (static_cast<int64_t>(sms) * 16 + a.groups - 1) / a.groups;
  if (shares > tiles) shares = tiles;
  if (shares < 1) shares = 1;
  const dim3 grid(static_cast<unsigned>(shares), static_cast<unsigned>(a.groups));
  if (a.beams <= 4)
    move_kernel<4><<<grid, kMoveThreads, 0, stream>>>(a);
  else if (a.beams <= 8)
    move_kernel<8><<<grid, kMoveThreads, 0, stream>>>(a);
  else if (a.beams <= 16)
    move_kernel<16><<<grid, kMoveThreads, 0, stream>>>(a);
  else if (a.beams <= 32)
    move_kernel<32><<<grid, kMoveThreads, 0, stream>>>(a);
  else
    move_kernel<64><<<grid, kMoveThreads, 0, stream>>>(a);
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
  for (int32_t k = 0; k < count; ++k) {  // every descriptor is checked before the first launch
    if (tensors[k].rows != tensors[0].rows) return fail(XG_EINVAL, "the tensors of a call have the same number of rows");
    if (tensors[k].rows < (rows ? 0 : static_cast<int64_t>(groups) * beams) || tensors[k].rows > 0x7fffffff)
      return fail(XG_EINVAL, "the tensors need one row per beam");
    MoveTensor m{};
    bool empty = false;
    if (int rc = describe(tensors[k], lengths != nullptr, beams, &m, &empty)) return rc;
  }
  MoveArgs a{};
  a.groups = groups;
  a.beams = beams;
  a.rows = tensors[0].rows;
  a.parents = parents;
  a.lengths = lengths;
  a.row_of = rows;
  int64_t units = 0;
  for (int32_t k = 0; k < count; ++k) {
    bool empty = false;
    MoveTensor& m = a.tensors[a.count];
    if (int rc = describe(tensors[k], lengths != nullptr, beams, &m, &empty)) return rc;
    if (!empty) {
      units += static_cast<int64_t>(m.size1) * m.size2 * m.size3;
      ++a.count;
    }
    if (a.count == kMoveTensors || (k + 1 == count && a.count > 0)) {
      if (int rc = launch_moves(a, units, stream)) return rc;
      a.count = 0;
      units = 0;
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
  a.segment = 32;
  a.window = kTraceBytes / 2 / beams;
  if (a.window > steps) a.window = steps;
  const int32_t segments = (a.window + a.segment - 1) / a.segment;
  const int32_t bytes = 2 * a.window * beams + 2 * segments * beams + beams;
  static std::atomic<bool> allowed[kDevices];
  if (int rc = allow_shared(reinterpret_cast<const void*>(trace_kernel), kTraceBytes + kTraceBytes / 16 + 1024, allowed)) return rc;
  trace_kernel<<<static_cast<unsigned>(groups), kTraceThreads, static_cast<size_t>(bytes),
                 reinterpret_cast<cudaStream_t>(stream)>>>(a);
  XG_BEAM_CUDA(cudaGetLastError(), "beam sequences kernel");
  return XG_OK;
}
