// libasap router: the top-k choice of an attention rank's MoE layer in the form asap_dispatch takes, its gradient, and
// the balance loss over the choice with per-expert counts.  The reference takes ids and weights from SGLang's top-k
// (python/sgl_asap_plugin/srt/layers/moe/ep_moe/layer.py:83-94 receives topk_output).
//
// One warp per token; lane l holds experts [l V, l V + V) in registers (V = 1 .. 32, at most 1024 experts), so a row is
// read once with 16-byte loads and the lowest lane of a tie has the lowest expert.
#include <cuda_fp16.h>

#include "common.cuh"

namespace asap {

int sm_count();

namespace route {

enum DType { kF32 = 0, kBf16 = 1, kF16 = 2 };
constexpr int kWarps = 8;         // tokens that a block works on at a time
constexpr int kRouteBlocks = 4;  // blocks of the router on an SM

__device__ __forceinline__ float to_float(uint16_t b, int dt) {
  if (dt == kBf16) return __uint_as_float((uint32_t)b << 16);
  return __half2float(__ushort_as_half(b));
}
__device__ __forceinline__ float load1(const void* row, int64_t e, int dt) {
  if (dt == kF32) return reinterpret_cast<const float*>(row)[e];
  return to_float(reinterpret_cast<const uint16_t*>(row)[e], dt);
}

// This lane's V values of a row of E; `fill` behind the row's end.  vec: rows start on 16-byte boundaries.
template <int V>
__device__ __forceinline__ void load_row(const void* row, int E, int dt, bool vec, int lane, float fill, float (&v)[V]) {
  const int e0 = lane * V;
  if (vec && e0 + V <= E) {
    if (dt == kF32) {
      const float* p = reinterpret_cast<const float*>(row) + e0;
      if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const float4 f = *reinterpret_cast<const float4*>(p + i);
          v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = p[i];
      }
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + e0;
      if constexpr (V >= 8) {
#pragma unroll
        for (int i = 0; i < V; i += 8) {
          const uint4 u = *reinterpret_cast<const uint4*>(p + i);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[i + 2 * j] = to_float((uint16_t)(w[j] & 0xffff), dt);
            v[i + 2 * j + 1] = to_float((uint16_t)(w[j] >> 16), dt);
          }
        }
      } else if constexpr (V >= 2) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(p + i);
          v[i] = to_float((uint16_t)(w & 0xffff), dt);
          v[i + 1] = to_float((uint16_t)(w >> 16), dt);
        }
      } else {
        v[0] = to_float(p[0], dt);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = e0 + i < E ? load1(row, e0 + i, dt) : fill;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int dt) {
  if (dt == kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int V>
__device__ __forceinline__ void store_row(void* row, int E, int dt, bool vec, int lane, const float (&v)[V]) {
  const int e0 = lane * V;
  if (vec && e0 + V <= E) {
    if (dt == kF32) {
      float* p = reinterpret_cast<float*>(row) + e0;
      if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4)
          *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = v[i];
      }
      return;
    }
    uint16_t* p = reinterpret_cast<uint16_t*>(row) + e0;
    if constexpr (V >= 8) {
#pragma unroll
      for (int i = 0; i < V; i += 8)
        *reinterpret_cast<uint4*>(p + i) = make_uint4(pack2(v[i], v[i + 1], dt), pack2(v[i + 2], v[i + 3], dt),
                                                      pack2(v[i + 4], v[i + 5], dt), pack2(v[i + 6], v[i + 7], dt));
      return;
    } else if constexpr (V >= 2) {
#pragma unroll
      for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(p + i) = pack2(v[i], v[i + 1], dt);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (e0 + i < E) {
      if (dt == kF32) reinterpret_cast<float*>(row)[e0 + i] = v[i];
      else reinterpret_cast<uint16_t*>(row)[e0 + i] = (uint16_t)(pack2(v[i], 0.f, dt) & 0xffff);
    }
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// Order-preserving unsigned keys (0 is free for "closed"; -0 and +0 share one key).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ double value_of(uint64_t k) {
  return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}
struct Args {
  const void* logits;
  int64_t ld;
  int32_t dtype, t, e, k, sigmoid, groups, top_groups, renorm, vec;
  // A group is a whole number of lanes, a power of two of them (or there is one group): the fast choice, whose shuffles
  // reduce a group.  Other groupings rank every row from the start in 64 bits, right and slow: 16384 x 160 in 8 groups
  // (V = 8, 20 experts a group) with a bias 101 us, in one group 16; 16384 x 256 in 8 groups 18.
  int32_t aligned_groups;
  int32_t group_log_lanes;
  float scale;
  const float* bias;         // NULL: none
  const int32_t* num_tokens;  // NULL: t
  int32_t* ids;
  float* weights;
};

// ---- the choice, fast form.  A lane sorts its V keys (a Batcher network of min / max); the low bits of a key give way
// to the expert's place in the lane, so that no index has to be carried along.  Every round takes the warp's best key (one
// redux) and the lane that held it moves on to its next.
//
// Keys rank as floats do.  Half-precision logits lose nothing to the place bits, and equal ones are a true tie.  Otherwise
// two keys that had to be compared may lie within the rounding of the scores, or differ in no bit that is left.  Then the
// scores of those few candidates are computed in 64 bits and ranked again; what that cannot settle makes the function
// return true, and the row is ranked exactly from the start.  (Both are kept small and rolled: a few rows of a call take
// them, and then wait for their instructions to be fetched.)
template <int V>
struct Place {
  static constexpr uint32_t MASK = V - 1;
};

template <int V>
__device__ __forceinline__ void sort_descending(uint32_t (&k)[V]) {
#pragma unroll
  for (int p = 1; p < V; p <<= 1)
#pragma unroll
    for (int q = p; q > 0; q >>= 1)
#pragma unroll
      for (int j = q % p; j + q < V; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
}

// key[i]: the key of expert lane * V + i with its place in the low bits; at most kClosed if the expert is closed.
// TIES: keys that differ in their place only are equal, and go to the lowest expert.  Else such keys are close, and so are
// two scores within tol + |score| (V + 2) 2^-23 of each other: tol for how the scores were computed (0: they are exact), V
// units in the last place for the place bits, two for the sum with the bias.
constexpr uint32_t kClosed = 0x007fffffu;  // the key of -inf
constexpr uint32_t kTwo = 0xc0000000u;     // the key of 2

// score + bias of one expert (a sigmoid), or its logit, in 64 bits
__device__ __noinline__ double exact_score(const Args& p, const void* row, int e) {
  const double x = (double)load1(row, e, p.dtype);
  return p.bias ? 1.0 / (1.0 + exp(-x)) + (double)p.bias[e] : x;
}

template <int V, bool TIES>
__device__ __forceinline__ bool choose(const Args& p, uint32_t (&key)[V], const void* row, int lane, bool& nan, int& my_id) {
  constexpr uint32_t MASK = Place<V>::MASK;
  constexpr float kUlps = (V + 2) * 1.1920929e-7f;
  const bool pairs = !TIES && p.bias;
  const float ninf = __uint_as_float(0xff800000u);
  const float tol = !p.bias ? 0.f : p.sigmoid ? 8e-7f : 4e-6f;
  const bool refinable = p.sigmoid || !p.bias;  // a softmax takes its whole row
  auto is_close = [&](uint32_t a, uint32_t b) {  // keys a >= b, both open
    const float x = value_of(a & ~MASK);
    // (negated: two infinities are close)
    return tol > 0.f ? !(x - value_of(b & ~MASK) >= tol + fabsf(x) * kUlps) : (a & ~MASK) == (b & ~MASK);
  };
  my_id = -1;
  sort_descending<V>(key);
  // two questions to the warp in one: a NaN in the row, a score above 2
  const uint32_t any = __reduce_or_sync(0xffffffffu, (nan ? 1u : 0u) | (key[0] > kTwo ? 2u : 0u));
  nan = any & 1u;
  if (p.groups > 1) {  // a group is an aligned run of lanes
    const int lanes = 1 << p.group_log_lanes;
    uint32_t best = key[0], second = V > 1 ? key[V > 1 ? 1 : 0] : 0u;
    for (int o = 1; o < lanes; o <<= 1) {
      const uint32_t ob = __shfl_xor_sync(0xffffffffu, best, o), os = __shfl_xor_sync(0xffffffffu, second, o);
      second = max(min(best, ob), max(second, os));
      best = max(best, ob);
    }
    best = __shfl_sync(0xffffffffu, best, lane * lanes);  // lane g: group g (lanes >= groups: unused)
    second = __shfl_sync(0xffffffffu, second, lane * lanes);
    const bool mine = lane < p.groups && best > kClosed;
    float score = mine ? value_of(best & ~MASK) : ninf;
    if (pairs && mine && second > kClosed) score += value_of(second & ~MASK);
    uint32_t k = mine ? key_of(score) : 0u, kept = 0, least = 0;
    for (int r = 0; r < p.top_groups; ++r) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, k);
      if (!m) break;
      const int g = __ffs(__ballot_sync(0xffffffffu, k == m)) - 1;
      kept |= 1u << g;
      if (lane == g) k = 0;
      least = m;
    }
    if (!TIES) {  // the least kept score against the best one dropped
      const uint32_t drop = __reduce_max_sync(0xffffffffu, k);
      bool close = drop && !pairs && is_close(least, drop);
      if (drop && pairs) {
        // A group's score is off by tol and the units of its two addends.  Unless one is above 2, they cannot cancel, and
        // are at most |score| + 4; then the order of the scores is in doubt only next to the border.
        const float x = value_of(least);
        close = (any & 2u) || !(x - value_of(drop) >= 2.f * (tol + (fabsf(x) + 4.f) * kUlps));
        if (close) {  // the least that a kept one can be against the most that a dropped one can
          const float size = fabsf(value_of(best & ~MASK)) + (second > kClosed ? fabsf(value_of(second & ~MASK)) : 0.f);
          const float off = tol + size * kUlps;
          const bool held = (kept >> lane) & 1u, sure = off < INFINITY;  // else it may be anything
          const uint32_t low = __reduce_min_sync(0xffffffffu, mine && held ? sure ? key_of(score - off) : 0u : 0xffffffffu);
          const uint32_t high = __reduce_max_sync(0xffffffffu, mine && !held ? sure ? key_of(score + off) : 0xffffffffu : 0u);
          close = low <= high;
        }
      }
      if (close) {
        // a lane's two best, in 64 bits, unless the third may be one of them
        const bool hard = V > 2 && key[V > 2 ? 2 : 0] > kClosed && is_close(key[V > 2 ? 1 : 0], key[V > 2 ? 2 : 0]);
        if (!refinable || __any_sync(0xffffffffu, hard)) return true;
        double a = -(double)INFINITY, b = a;
#pragma unroll 1
        for (int i = 0; i < (V > 1 ? 2 : 1); ++i) {
          const uint32_t x = i ? key[V > 1 ? 1 : 0] : key[0];
          const double d = x > kClosed ? exact_score(p, row, lane * V + (int)(MASK - (x & MASK))) : -(double)INFINITY;
          b = d > a ? a : d;
          a = d > a ? d : a;
        }
#pragma unroll 1
        for (int o = 1; o < lanes; o <<= 1) {
          const double oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
          b = fmax(fmin(a, oa), fmax(b, ob));
          a = fmax(a, oa);
        }
        a = __shfl_sync(0xffffffffu, a, lane * lanes);
        b = __shfl_sync(0xffffffffu, b, lane * lanes);
        if (pairs && b > -(double)INFINITY) a += b;
        int rank = 0;
#pragma unroll 1
        for (int g = 0; g < p.groups; ++g) {
          const double o = __shfl_sync(0xffffffffu, a, g);
          rank += o > a || (o == a && g < lane);
        }
        kept = __ballot_sync(0xffffffffu, mine && rank < p.top_groups);
      }
    }
    if (!((kept >> (lane >> p.group_log_lanes)) & 1u)) {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = 0;
    }
  }
  // lane j: the key taken in round j.  Beyond the k-th as long as the next one is close to the last.
  uint32_t mine = 0, prev = 0;
  int j = 0;
  for (;; ++j) {
    uint32_t m;
    int src, id;
    if (TIES) {
      if (j == p.k) break;
      m = __reduce_max_sync(0xffffffffu, key[0] & ~MASK);
      src = __ffs(__ballot_sync(0xffffffffu, (key[0] & ~MASK) == m)) - 1;
      id = src * V + (int)(MASK - (__shfl_sync(0xffffffffu, key[0], src) & MASK));
    } else {
      m = __reduce_max_sync(0xffffffffu, key[0]);
      if (j >= p.k) {
        if (m <= kClosed || !is_close(prev, m)) break;
        if (j == 32) return true;
      }
      src = __ffs(__ballot_sync(0xffffffffu, key[0] == m)) - 1;
      id = src * V + (int)(MASK - (m & MASK));
      prev = m;
    }
    if (lane == j) {
      mine = m;
      my_id = id;
    }
    const bool taken = lane == src;
#pragma unroll
    for (int i = 0; i + 1 < V; ++i) key[i] = taken ? key[i + 1] : key[i];
    key[V - 1] = taken ? 0u : key[V - 1];
  }
  if (mine <= kClosed) my_id = -1;
  if (!TIES) {
    const uint32_t before = __shfl_up_sync(0xffffffffu, mine, 1);
    if (__any_sync(0xffffffffu, lane > 0 && mine > kClosed && is_close(before, mine))) {
      if (!refinable) return true;
      const double d = my_id >= 0 ? exact_score(p, row, my_id) : -(double)INFINITY;
      int rank = 0, sorted = -1;
#pragma unroll 1
      for (int s = 0; s < j; ++s) {
        const double o = __shfl_sync(0xffffffffu, d, s);
        const int oid = __shfl_sync(0xffffffffu, my_id, s);
        rank += o > d || (o == d && (unsigned)oid < (unsigned)my_id);  // -1, no expert, ranks last
      }
#pragma unroll 1
      for (int s = 0; s < j; ++s) {
        const int r = __shfl_sync(0xffffffffu, rank, s), id = __shfl_sync(0xffffffffu, my_id, s);
        if (r == lane && id >= 0) sorted = id;
      }
      my_id = sorted;
    }
  }
  if (lane >= p.k) my_id = -1;
  return false;
}

// ---- the choice of one row in 64 bits, from memory, for any groups.  Rolled loops; a lane goes through its keys again for
// every group and every round.
template <int V>
__device__ __noinline__ int choose_exactly(const Args& p, const void* row, int lane) {
  const double ninf = -(double)INFINITY;
  double z = 0.0, top = ninf;
  if (p.bias && !p.sigmoid) {
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        const int e = lane * V + i;
        const double x = e < p.e ? (double)load1(row, e, p.dtype) : ninf;
        if (!pass) top = fmax(top, x);
        else if (x > ninf) z += exp(x - top);
      }
      if (!pass)
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    z = warp_sum(z);
  }
  uint64_t key[V];  // 0: closed
#pragma unroll 1
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    double x = e < p.e ? (double)load1(row, e, p.dtype) : ninf;
    const bool open = x > ninf;  // false for NaN
    if (p.bias && open) x = (p.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - top) / z) + (double)p.bias[e];
    key[i] = open && x > ninf ? key_of(x) : 0ull;
  }
  if (p.groups > 1) {
    const int size = p.e / p.groups;
    double score = ninf;  // lane g: group g
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      uint64_t a = 0, c = 0;
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        const int e = lane * V + i;
        const uint64_t x = e >= g * size && e < g * size + size ? key[i] : 0ull;
        c = x > a ? a : x > c ? x : c;
        a = x > a ? x : a;
      }
      const uint64_t m = warp_max(a);
      const uint32_t holders = __ballot_sync(0xffffffffu, a == m);
      const uint64_t rest = warp_max(a == m && lane == __ffs(holders) - 1 ? c : a);
      if (lane == g && m) score = value_of(m) + (p.bias && rest ? value_of(rest) : 0.0);
    }
    int rank = 0;
#pragma unroll 1
    for (int g = 0; g < p.groups; ++g) {
      const double o = __shfl_sync(0xffffffffu, score, g);
      rank += o > score || (o == score && g < lane);
    }
    const uint32_t kept = __ballot_sync(0xffffffffu, lane < p.groups && score > ninf && rank < p.top_groups);
#pragma unroll 1
    for (int i = 0; i < V; ++i)
      if (lane * V + i < p.e && !((kept >> ((lane * V + i) / size)) & 1u)) key[i] = 0;
  }
  int my_id = -1;
#pragma unroll 1
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll 1
    for (int i = 0; i < V; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const uint64_t m = warp_max(best);
    if (!m) break;
    const int src = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
    const int id = __shfl_sync(0xffffffffu, lane * V + at, src);
    if (lane == j) my_id = id;
    if (lane == src) key[at] = 0;
  }
  return my_id;
}

__device__ __forceinline__ float rcp_approx(float x) {  // within 1 ulp; 0 for infinity
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float exp_approx(float x) {  // within 2 + |x| / 2^24 * 1.5 ulp
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// Without a bias the scores rank as the logits do, so the choice compares logits.  With one it compares score + bias in
// fp32, and ranks a row with two candidates closer than the fp32 error (one in a thousand rows) again in 64 bits.  The
// bounds: a sigmoid is off by at most 4 * 10^-7 (fast exponential 2^-22 + |x| 2^-23.2 relative, times a slope of at most
// s (1 - s) <= 1/4; a sum; a reciprocal within 1 ulp), a softmax by 2 * 10^-6 (a sum of up to 1024 terms), and a pair by
// twice that.
//
// Bound by issue slots (68%): 860 instructions of a warp per token at 256 experts, top 8 of 4 of 8 groups with a bias (an
// exponential and a reciprocal for each of a lane's experts, sorting them, a round of 20 per place).
// TIES: half-precision logits without a bias
template <int V, bool TIES>
__global__ void __launch_bounds__(32 * kWarps, V <= 8 ? kRouteBlocks : 2) route_kernel(const __grid_constant__ Args p) {
  constexpr uint32_t MASK = Place<V>::MASK;
  const int lane = threadIdx.x & 31;
  const int step = gridDim.x * kWarps;
  const float ninf = __uint_as_float(0xff800000u);
  const int n = p.num_tokens ? min(max(*p.num_tokens, 0), p.t) : p.t;
  auto row_of = [&](int t) {
    return reinterpret_cast<const void*>(reinterpret_cast<const uint8_t*>(p.logits) +
                                         (int64_t)t * p.ld * (p.dtype == kF32 ? 4 : 2));
  };
  int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
  float next[V];
  if (t < n) load_row<V>(row_of(t), p.e, p.dtype, p.vec, lane, ninf, next);
  for (; t < p.t; t += step) {
    int32_t* ids = p.ids + (int64_t)t * p.k;
    float* weights = p.weights + (int64_t)t * p.k;
    if (t >= n) {
      if (lane < p.k) {
        ids[lane] = -1;
        weights[lane] = 0.f;
      }
      continue;
    }
    const void* row = row_of(t);
    float l[V];
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = next[i];
    if (t + step < n) load_row<V>(row_of(t + step), p.e, p.dtype, p.vec, lane, ninf, next);
    bool nan = false;
    float top = ninf, z = 1.f;
#pragma unroll
    for (int i = 0; i < V; ++i) nan |= l[i] != l[i];
    if (!p.sigmoid) {
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, l[i]);
      top = warp_max(top);
      z = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (l[i] > ninf) z += expf(l[i] - top);
      z = warp_sum(z);
    }
    int id;
    uint32_t key[V];
    bool unsure = !p.aligned_groups;
    if (unsure) {
      nan = __any_sync(0xffffffffu, nan);
    } else {
      float b[V];
      const float rz = 1.f / z;
      if (!TIES && p.bias)
        load_row<V>(p.bias, p.e, kF32, (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0, lane, ninf, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float x = l[i];
        if (!TIES && p.bias) x = (p.sigmoid ? rcp_approx(1.f + exp_approx(-x)) : expf(x - top) * rz) + b[i];
        x = fmaxf(l[i] > ninf ? x : ninf, ninf);  // NaN is closed
        key[i] = (key_of(x) & ~MASK) | (MASK - i);
      }
      unsure = choose<V, TIES>(p, key, row, lane, nan, id);
    }
    if (unsure) id = choose_exactly<V>(p, row, lane);
    float s = 0.f;
    if (id >= 0) {
      const float x = load1(row, id, p.dtype);
      s = p.sigmoid ? 1.f / (1.f + expf(-x)) : expf(x - top) / z;
    }
    const float sum = p.renorm ? warp_sum(s) + 1e-20f : 1.f;
    if (lane < p.k) {
      ids[lane] = id;
      weights[lane] = nan ? __uint_as_float(0x7fc00000u) : p.scale * (s / sum);
    }
  }
}

// ------------------------------------------------------------------ gradient of the weights to the logits
// w_j = c s_j / N with N = sum of the selected s + 1e-20 (1 without renormalisation).  ds_j = c / N (g_j - [renorm]
// sum_i g_i s_i / N) on the selected experts; sigmoid: dl_j = s_j (1 - s_j) ds_j.  softmax: dl_e = s_e (ds_e - sum_i
// ds_i s_i) for every e; after renormalisation that sum is c (sum g s) / N (1 - S / N), nothing unless S is of the size
// of 1e-20, which only a bias can bring about: `dense` asks for the row's softmax.  Every form reads the row, for a NaN in
// it: such a row's weights are NaN, so its gradient is NaN too, all of it.
struct BackArgs {
  const void* logits;
  int64_t ld;
  int32_t dtype, t, e, k, sigmoid, dense, renorm, vec, out_vec;
  float scale;
  const int32_t* ids;
  const float* grad;
  void* out;  // [t, e] of the logits' type
};

template <int V>
__global__ void __launch_bounds__(32 * kWarps) route_back_kernel(const __grid_constant__ BackArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (t >= p.t) return;
  const int size = p.dtype == kF32 ? 4 : 2;
  const void* row = reinterpret_cast<const uint8_t*>(p.logits) + t * p.ld * size;
  const float ninf = __uint_as_float(0xff800000u);
  int id = -1;
  float g = 0.f, x = ninf;
  if (lane < p.k) {
    id = p.ids[t * p.k + lane];
    if (id < 0 || id >= p.e) id = -1;
    if (id >= 0) {
      g = p.grad[t * p.k + lane];
      x = load1(row, id, p.dtype);
    }
  }
  float s, d[V];
  if (!__any_sync(0xffffffffu, id >= 0)) {  // a padding row, or none left: nothing of its logits, which may be NaN, counts
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = 0.f;
    store_row<V>(reinterpret_cast<uint8_t*>(p.out) + t * p.e * size, p.e, p.dtype, p.out_vec, lane, d);
    return;
  }
  load_row<V>(row, p.e, p.dtype, p.vec, lane, ninf, d);
  bool nan = false;
#pragma unroll
  for (int i = 0; i < V; ++i) nan |= d[i] != d[i];
  nan = __any_sync(0xffffffffu, nan);
  if (p.sigmoid) {
    s = id >= 0 ? 1.f / (1.f + expf(-x)) : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = 0.f;
  } else {
    float z = 0.f, top;
    if (p.dense) {
      top = ninf;
#pragma unroll
      for (int i = 0; i < V; ++i) top = fmaxf(top, d[i]);
      top = warp_max(top);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = d[i] == ninf ? 0.f : expf(d[i] - top);
        z += d[i];
      }
      z = warp_sum(z);
      z = z > 0.f ? 1.f / z : 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] *= z;
      s = id >= 0 ? expf(x - top) * z : 0.f;
    } else {  // relative to the selected experts: the common factor cancels
      top = warp_max(x);
      s = id >= 0 ? expf(x - top) : 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = 0.f;
    }
  }
  const float n = p.renorm ? warp_sum(s) + (p.sigmoid || p.dense ? 1e-20f : 0.f) : 1.f;
  const float gs = p.renorm ? warp_sum(g * s) / n : 0.f;
  float ds = id >= 0 ? p.scale / n * (g - gs) : 0.f;
  float mine;  // this lane's selected expert: its gradient beyond the dense term
  if (p.sigmoid) {
    mine = id >= 0 ? ds * s * (1.f / (1.f + expf(x))) : 0.f;  // 1 - s without cancellation
  } else {
    const float dot = p.dense ? warp_sum(ds * s) : 0.f;
    mine = ds * s;
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = p.dense ? -d[i] * dot : 0.f;
  }
  for (int j = 0; j < p.k; ++j) {
    const int e = __shfl_sync(0xffffffffu, id, j);
    const float v = __shfl_sync(0xffffffffu, mine, j);
    if (e >= 0 && e / V == lane) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e % V == i) d[i] += v;
    }
  }
  if (nan) {
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = __uint_as_float(0x7fc00000u);
  }
  store_row<V>(reinterpret_cast<uint8_t*>(p.out) + t * p.e * size, p.e, p.dtype, p.out_vec, lane, d);
}

// ------------------------------------------------------------------ balance loss
// Over the sequences s with n_s > 0 live tokens (a token is live when it has an id), S' of them:
//   L = coef / S' sum_s sum_e f_se P_se,  f_se = E / (k n_s) c_se,  P_se = 1 / n_s sum_t p_te,
// c the counts, p the row's softmax, or its sigmoids normalised to sum 1.  With a_se = coef / S' E / (k n_s^2) c_se that
// is a plain sum over tokens, L = sum_t sum_e a_se p_te, and the gradient is dl_te = p_te (a_se - sum_i a_si p_ti),
// times 1 - sigmoid(l_te) for sigmoids: once the counts are there, each direction is one pass over the rows, and no sum
// of probabilities over tokens is kept.
struct BalanceArgs {
  const void* logits;
  int64_t ld;
  int32_t dtype, t, e, k, sigmoid, seqs, vec, out_vec;
  float coef;
  const int32_t* ids;
  const int32_t* cu;   // [seqs + 1], NULL: one sequence of t tokens
  int32_t* counts;     // [seqs, e]
  int32_t* live;       // [seqs]
  uint32_t* ticket;    // [2] blocks that have finished counting / adding
  float* factor;       // [seqs] coef / S' E / (k n_s^2)
  int32_t* row_seq;    // [t] the sequence of a live token, else -1
  double* partial;     // [grid]
  float* loss;
  const float* grad;   // d loss, scalar
  void* out;
};

// the sequence of token t, or -1 (before the first or behind the last)
__device__ __forceinline__ int seq_of(const int32_t* cu, int seqs, int64_t t) {
  if (!cu) return 0;
  if (t < cu[0]) return -1;
  int lo = 0, hi = seqs;  // first s with cu[s + 1] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo < seqs ? lo : -1;
}

constexpr int kCountRows = 64;  // tokens per block
constexpr int kCountThreads = 128;
constexpr int kCountSeqs = 1024;  // up to here the offsets are searched in shared memory
// Counts and live tokens per sequence, each token's sequence (-1: not live) for the passes over the logits, and, by the
// block that finishes last, the factor of each sequence's counts in a_se.
__global__ void __launch_bounds__(kCountThreads) balance_count_kernel(const __grid_constant__ BalanceArgs p) {
  extern __shared__ int32_t hist[];  // [e + 1]: the counts of the block's first sequence, and its live tokens
  __shared__ int32_t s_cu[kCountSeqs + 1], s_seq[kCountRows], s_live[kCountRows];
  __shared__ bool s_last;
  __shared__ int s_filled;
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)blockIdx.x * kCountRows;
  const int rows = (int)min((int64_t)kCountRows, p.t - t0), n = rows * p.k;
  const int32_t* ids = p.ids + t0 * p.k;
  for (int i = tid; i <= p.e; i += kCountThreads) hist[i] = 0;
  const bool staged = p.cu && p.seqs <= kCountSeqs;
  if (staged)
    for (int i = tid; i <= p.seqs; i += kCountThreads) s_cu[i] = p.cu[i];
  if (tid < kCountRows) s_live[tid] = 0;
  __syncthreads();
  if (tid < rows) s_seq[tid] = seq_of(staged ? s_cu : p.cu, p.seqs, t0 + tid);
  __syncthreads();
  const int first = s_seq[0];
#pragma unroll 4
  for (int i = tid; i < n; i += kCountThreads) {
    const int e = ids[i], r = i / p.k, s = s_seq[r];
    if (e < 0 || e >= p.e || s < 0) continue;
    s_live[r] = 1;
    atomicAdd(s == first ? &hist[e] : &p.counts[(int64_t)s * p.e + e], 1);
  }
  __syncthreads();
  if (p.live && tid < rows) {
    const int s = s_live[tid] ? s_seq[tid] : -1;
    p.row_seq[t0 + tid] = s;
    if (s >= 0) atomicAdd(s == first ? &hist[p.e] : &p.live[s], 1);
  }
  __syncthreads();
  if (first >= 0)
    for (int i = tid; i <= p.e; i += kCountThreads)
      if (hist[i]) {
        if (i < p.e) atomicAdd(&p.counts[(int64_t)first * p.e + i], hist[i]);
        else if (p.live) atomicAdd(&p.live[first], hist[i]);
      }
  if (!p.live) return;  // counts alone
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    s_last = atomicAdd(&p.ticket[0], 1u) == gridDim.x - 1;
    s_filled = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  int filled = 0;
  for (int s = tid; s < p.seqs; s += kCountThreads) filled += __ldcg(&p.live[s]) > 0;
  filled = __reduce_add_sync(0xffffffffu, filled);
  if ((tid & 31) == 0) atomicAdd(&s_filled, filled);
  __syncthreads();
  const float base = p.coef / (float)max(s_filled, 1) * ((float)p.e / (float)p.k);
  for (int s = tid; s < p.seqs; s += kCountThreads) {
    const float live = (float)max(__ldcg(&p.live[s]), 1);
    p.factor[s] = base / (live * live);
  }
}

// p_e of a row, and q_e = 1 - sigmoid(l_e) with sigmoids, whose quotients are approximate (2 units in the last place, as the
// exponential before them).  A row of sigmoids whose largest logit is negative is scaled by
// e^-top, so that its values do not underflow before they are normalised.
template <int V>
__device__ __forceinline__ void row_probabilities(bool sigmoid, float (&l)[V], float (&p)[V], float (&q)[V]) {
  const float ninf = __uint_as_float(0xff800000u);
  float top = ninf, z = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) top = fmaxf(top, l[i]);
  top = warp_max(top);
  if (!sigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = l[i] == ninf ? 0.f : expf(l[i] - top);
  } else if (top >= 0.f) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = fminf(expf(-l[i]), 1e30f);  // sigmoid = 1 / (1 + x), 1 - sigmoid = x / (1 + x)
      const float s = __fdividef(1.f, 1.f + x);
      p[i] = l[i] == ninf ? 0.f : l[i] != l[i] ? l[i] : s;
      q[i] = x * s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      q[i] = __fdividef(1.f, 1.f + expf(l[i]));
      p[i] = l[i] == ninf ? 0.f : expf(l[i] - top) * q[i];
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) z += p[i];
  z = warp_sum(z);
  const float r = z > 0.f ? 1.f / z : (z != z ? z : 0.f);
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] *= r;
}

// A warp takes a run of tokens, so that the sequence it is in, and that sequence's a_e, change rarely; the next token's
// logits are on their way while one is worked on.
template <int V, bool BACK>
__global__ void __launch_bounds__(32 * kWarps, V <= 8 ? 4 : 2) balance_kernel(const __grid_constant__ BalanceArgs p) {
  __shared__ double s_sum[kWarps];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int size = p.dtype == kF32 ? 4 : 2;
  const float ninf = __uint_as_float(0xff800000u);
  const int64_t per_warp = (p.t + (int64_t)gridDim.x * kWarps - 1) / ((int64_t)gridDim.x * kWarps);
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + warp) * per_warp, t1 = min((int64_t)p.t, t0 + per_warp);
  auto row = [&](int64_t t) { return reinterpret_cast<const uint8_t*>(p.logits) + t * p.ld * size; };
  float next[V];
  int next_seq = -1;
  if (t0 < t1) {
    load_row<V>(row(t0), p.e, p.dtype, p.vec, lane, ninf, next);
    next_seq = p.row_seq[t0];
  }
  const float grad = BACK ? *p.grad : 1.f;
  double sum = 0.0;
  int seq = -1;
  float a[V];
  for (int64_t t = t0; t < t1; ++t) {
    float l[V];
    const int s = next_seq;
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = next[i];
    if (t + 1 < t1) {
      load_row<V>(row(t + 1), p.e, p.dtype, p.vec, lane, ninf, next);
      next_seq = p.row_seq[t + 1];
    }
    float d[V];
    if (s >= 0) {
      if (s != seq) {
        seq = s;
        const float f = p.factor[s] * grad;
        const int32_t* counts = p.counts + (int64_t)s * p.e + lane * V;
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = lane * V + i < p.e ? f * (float)counts[i] : 0.f;
      }
      float pr[V], q[V], dot = 0.f;
      row_probabilities<V>(p.sigmoid != 0, l, pr, q);
#pragma unroll
      for (int i = 0; i < V; ++i) dot += a[i] * pr[i];
      dot = warp_sum(dot);
      if constexpr (BACK) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[i] = pr[i] * (a[i] - dot);
          if (p.sigmoid) d[i] *= q[i];
        }
      } else {
        sum += (double)dot;
      }
    } else if constexpr (BACK) {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = 0.f;
    }
    if constexpr (BACK)
      store_row<V>(reinterpret_cast<uint8_t*>(p.out) + t * p.e * size, p.e, p.dtype, p.out_vec, lane, d);
  }
  if constexpr (!BACK) {
    // block sums, added in block order by the block that finishes last: the same bits every time
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      double b = 0.0;
      for (int w = 0; w < kWarps; ++w) b += s_sum[w];
      p.partial[blockIdx.x] = b;
      __threadfence();
      s_last = atomicAdd(&p.ticket[1], 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (s_last && warp == 0) {
      __threadfence();
      double b = 0.0;
      for (int i = lane; i < (int)gridDim.x; i += 32) b += __ldcg(&p.partial[i]);
      b = warp_sum(b);
      if (lane == 0) *p.loss = (float)b;
    }
  }
}

// A few tokens in one block and one launch: the counts, sequences and factors as balance_count_kernel leaves them, and the
// loss.  Against a memset, the counts and the loss the caller saves two launches, 21 us of its time for 25; on the GPU (us,
// here / there) it wins while one block keeps up:
//   16 experts:  16 tokens  3.8 /  9.7, 192  7.8 / 11.1, 320 10.7 / 12.1, 384 12.1 / 11.9, 512 15.0 / 11.5, 768 20.9 / 11.8
//   64:          16 tokens  4.2 / 11.2, 128  6.7 / 11.6, 256  9.9 / 12.4, 384 13.2 / 12.4, 512 16.5 / 12.4
//   256:         16 tokens  5.1 / 11.9,  64  8.2 / 13.1, 128 12.9 / 13.0, 192 17.6 / 14.0
//   1000:        16 tokens 17.3 / 19.3,  32 29.2 / 20.3
// Taken where what the GPU loses is no more than the 4 us that the caller saves, for every number of experts: tokens x V up
// to 512 (the widest margin is left with 64 to 512 experts, the least with 16 and 512 tokens, where a captured graph loses
// 3.5 us and an eager call gains 4).
constexpr int kSmallWarps = 32, kSmallTokens = 512, kSmallCounts = 4096;  // tokens x V; sequences x experts
template <int V>
__global__ void __launch_bounds__(32 * kSmallWarps) balance_small_kernel(const __grid_constant__ BalanceArgs p) {
  __shared__ int32_t s_counts[kSmallCounts], s_live[kSmallCounts], s_seq[kSmallTokens];  // 34 KB
  __shared__ double s_sum[kSmallWarps];
  __shared__ int s_filled;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int size = p.dtype == kF32 ? 4 : 2;
  const float ninf = __uint_as_float(0xff800000u);
  const int cells = p.seqs * p.e;
  for (int i = tid; i < cells; i += 32 * kSmallWarps) s_counts[i] = 0;
  for (int i = tid; i < p.seqs; i += 32 * kSmallWarps) s_live[i] = 0;
  if (tid == 0) s_filled = 0;
  __syncthreads();
  for (int t = tid; t < p.t; t += 32 * kSmallWarps) {
    const int s = seq_of(p.cu, p.seqs, t);
    bool any = false;
    if (s >= 0)
      for (int j = 0; j < p.k; ++j) {
        const int e = p.ids[(int64_t)t * p.k + j];
        if (e < 0 || e >= p.e) continue;
        any = true;
        atomicAdd(&s_counts[s * p.e + e], 1);
      }
    if (any) atomicAdd(&s_live[s], 1);
    s_seq[t] = any ? s : -1;
    p.row_seq[t] = any ? s : -1;
  }
  __syncthreads();
  int filled = 0;
  for (int s = tid; s < p.seqs; s += 32 * kSmallWarps) filled += s_live[s] > 0;
  filled = __reduce_add_sync(0xffffffffu, filled);
  if (lane == 0) atomicAdd(&s_filled, filled);
  __syncthreads();
  const float base = p.coef / (float)max(s_filled, 1) * ((float)p.e / (float)p.k);
  for (int s = tid; s < p.seqs; s += 32 * kSmallWarps) {
    const float live = (float)max(s_live[s], 1);
    p.factor[s] = base / (live * live);
    p.live[s] = s_live[s];
  }
  for (int i = tid; i < cells; i += 32 * kSmallWarps) p.counts[i] = s_counts[i];
  double sum = 0.0;
  constexpr int U = V <= 2 ? 4 : V <= 4 ? 2 : 1;  // rows on their way at once
  for (int t0 = warp; t0 < p.t; t0 += U * kSmallWarps) {
    float l[U][V];
    int seq[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * kSmallWarps;
      seq[u] = t < p.t ? s_seq[t] : -1;
      if (seq[u] >= 0)
        load_row<V>(reinterpret_cast<const uint8_t*>(p.logits) + (int64_t)t * p.ld * size, p.e, p.dtype, p.vec, lane, ninf,
                    l[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (seq[u] < 0) continue;
      float pr[V], q[V], dot = 0.f;
      row_probabilities<V>(p.sigmoid != 0, l[u], pr, q);
      const float live = (float)s_live[seq[u]], f = base / (live * live);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (lane * V + i < p.e) dot += f * (float)s_counts[seq[u] * p.e + lane * V + i] * pr[i];
      sum += (double)warp_sum(dot);
    }
  }
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    double b = 0.0;
    for (int w = 0; w < kSmallWarps; ++w) b += s_sum[w];
    *p.loss = (float)b;
  }
}

// ------------------------------------------------------------------ host side
static int per_lane(int e) {  // V
  int v = 1;
  while (32 * v < e) v *= 2;
  return v;
}
template <template <int> class F, typename A>
static void by_experts(int e, const A& a, int grid, cudaStream_t st) {
  switch (per_lane(e)) {
    case 1: return F<1>::run(a, grid, st);
    case 2: return F<2>::run(a, grid, st);
    case 4: return F<4>::run(a, grid, st);
    case 8: return F<8>::run(a, grid, st);
    case 16: return F<16>::run(a, grid, st);
    default: return F<32>::run(a, grid, st);
  }
}
template <int V>
struct Forward {
  static void run(const Args& a, int grid, cudaStream_t st) {
    if (!a.bias && a.dtype != kF32) route_kernel<V, true><<<grid, 32 * kWarps, 0, st>>>(a);
    else route_kernel<V, false><<<grid, 32 * kWarps, 0, st>>>(a);
  }
};
template <int V>
struct Backward {
  static void run(const BackArgs& a, int grid, cudaStream_t st) { route_back_kernel<V><<<grid, 32 * kWarps, 0, st>>>(a); }
};
template <int V>
struct Loss {
  static void run(const BalanceArgs& a, int grid, cudaStream_t st) {
    balance_kernel<V, false><<<grid, 32 * kWarps, 0, st>>>(a);
  }
};
template <int V>
struct LossSmall {
  static void run(const BalanceArgs& a, int, cudaStream_t st) { balance_small_kernel<V><<<1, 32 * kSmallWarps, 0, st>>>(a); }
};
template <int V>
struct LossBack {
  static void run(const BalanceArgs& a, int grid, cudaStream_t st) {
    balance_kernel<V, true><<<grid, 32 * kWarps, 0, st>>>(a);
  }
};

static int check_logits(const char* fn, uint64_t logits, int64_t ld, int32_t dtype, int32_t t, int32_t e, int32_t k) {
  if (t < 1 || e < 1 || e > ASAP_ROUTE_MAX_EXPERTS || k < 1 || k > ASAP_ROUTE_MAX_TOPK || k > e || t > (1 << 24)) {
    set_error("%s: need 1 to %d tokens, 1 <= k <= %d, k <= experts <= %d (got %d tokens, k = %d, %d experts)", fn, 1 << 24,
              ASAP_ROUTE_MAX_TOPK, ASAP_ROUTE_MAX_EXPERTS, t, k, e);
    return ASAP_EINVAL;
  }
  if (dtype < 0 || dtype > 2 || !logits || (logits & (dtype ? 1 : 3)) || ld < e) {
    set_error("%s: logits must be fp32 (0), bf16 (1) or fp16 (2), aligned to their type, with a row stride of at least "
              "%d (got type %d, stride %lld)", fn, e, dtype, (long long)ld);
    return ASAP_EINVAL;
  }
  return ASAP_OK;
}
static bool rows_16(uint64_t base, int64_t ld, int32_t dtype) {
  return (base & 15) == 0 && (ld * (dtype ? 2 : 4)) % 16 == 0;
}

struct BalanceWs {
  uint64_t ticket, zeroed, factor, row_seq, partial, bytes;
};
static BalanceWs balance_ws(int64_t t, int64_t seqs) {
  BalanceWs w;
  w.ticket = 4 * seqs;     // after the live tokens
  w.zeroed = w.ticket + 8;  // live tokens and tickets start at 0
  w.factor = w.zeroed;
  w.row_seq = w.factor + 4 * seqs;
  w.partial = align_up(w.row_seq + 4 * t, 8);
  w.bytes = w.partial + 8ull * 4 * sm_count();
  return w;
}
static int balance_grid(int32_t t) {
  const int64_t blocks = ((int64_t)t + kWarps - 1) / kWarps, cap = 4ll * sm_count();
  return (int)(blocks < cap ? blocks : cap);
}

static int balance_args(const char* fn, BalanceArgs& a, const asap_balance_t* b, uint64_t ws, uint64_t ws_bytes) {
  if (!b) {
    set_error("%s: NULL argument", fn);
    return ASAP_EINVAL;
  }
  if (int rc = check_logits(fn, b->logits, b->ld, b->dtype, b->t, b->e, b->k)) return rc;
  if (!b->counts || (b->counts & 3) || !b->ids || (b->ids & 3) || b->seqs < 1 || b->seqs > (1 << 20) || (!b->cu_seqlens && b->seqs != 1) ||
      (b->cu_seqlens & 3)) {
    set_error("%s: need ids, counts and 1 to %d sequences (one without offsets), got %d", fn, 1 << 20, b->seqs);
    return ASAP_EINVAL;
  }
  const BalanceWs w = balance_ws(b->t, b->seqs);
  if (!ws || (ws & 7) || ws_bytes < w.bytes) {
    set_error("%s: the workspace must be 8-byte aligned and hold %llu bytes (got %llu)", fn, (unsigned long long)w.bytes,
              (unsigned long long)ws_bytes);
    return ASAP_EINVAL;
  }
  a.logits = (const void*)b->logits;
  a.ld = b->ld;
  a.dtype = b->dtype;
  a.t = b->t;
  a.e = b->e;
  a.k = b->k;
  a.sigmoid = b->sigmoid;
  a.seqs = b->seqs;
  a.vec = rows_16(b->logits, b->ld, b->dtype);
  a.coef = b->coef;
  a.ids = (const int32_t*)b->ids;
  a.cu = (const int32_t*)b->cu_seqlens;
  a.counts = (int32_t*)b->counts;
  a.live = (int32_t*)ws;
  a.ticket = (uint32_t*)(ws + w.ticket);
  a.factor = (float*)(ws + w.factor);
  a.row_seq = (int32_t*)(ws + w.row_seq);
  a.partial = (double*)(ws + w.partial);
  return ASAP_OK;
}

}  // namespace route
}  // namespace asap

using namespace asap;

extern "C" {

int asap_route(const asap_route_t* r, uint64_t ids, uint64_t weights, void* stream) {
  if (!r) {
    set_error("asap_route: NULL argument");
    return ASAP_EINVAL;
  }
  if (int rc = route::check_logits("asap_route", r->logits, r->ld, r->dtype, r->t, r->e, r->k)) return rc;
  if (r->groups < 1 || r->groups > 32 || r->e % r->groups || r->top_groups < 1 || r->top_groups > r->groups) {
    set_error("asap_route: %d groups of %d experts, %d kept: need 1 to 32 equal groups and 1 <= kept <= groups",
              r->groups, r->e, r->top_groups);
    return ASAP_EINVAL;
  }
  if (!ids || (ids & 3) || !weights || (weights & 3) || (r->bias & 3) || (r->num_tokens & 3)) {
    set_error("asap_route: ids and weights must be non-NULL, and every pointer 4-byte aligned");
    return ASAP_EINVAL;
  }
  route::Args a{};
  a.logits = (const void*)r->logits;
  a.ld = r->ld;
  a.dtype = r->dtype;
  a.t = r->t;
  a.e = r->e;
  a.k = r->k;
  a.sigmoid = r->sigmoid;
  a.groups = r->top_groups == r->groups ? 1 : r->groups;  // every group kept: no limit
  a.top_groups = r->top_groups;
  const int v = route::per_lane(r->e), lanes = r->e / a.groups / v;
  while ((2 << a.group_log_lanes) <= lanes) ++a.group_log_lanes;
  a.aligned_groups = a.groups == 1 || (r->e % (a.groups * v) == 0 && (lanes & (lanes - 1)) == 0);
  a.renorm = r->renormalize;
  a.vec = route::rows_16(r->logits, r->ld, r->dtype);
  a.scale = r->scale;
  a.bias = (const float*)r->bias;
  a.num_tokens = (const int32_t*)r->num_tokens;
  a.ids = (int32_t*)ids;
  a.weights = (float*)weights;
  const int blocks = (r->t + route::kWarps - 1) / route::kWarps, cap = route::kRouteBlocks * sm_count();
  route::by_experts<route::Forward>(r->e, a, blocks < cap ? blocks : cap, (cudaStream_t)stream);
  ASAP_CHECK_LAUNCH("route_kernel");
  return ASAP_OK;
}

int asap_route_backward(const asap_route_t* r, uint64_t ids, uint64_t grad_weights, uint64_t grad_logits,
                        void* stream) {
  if (!r) {
    set_error("asap_route_backward: NULL argument");
    return ASAP_EINVAL;
  }
  if (int rc = route::check_logits("asap_route_backward", r->logits, r->ld, r->dtype, r->t, r->e, r->k)) return rc;
  if (!ids || (ids & 3) || !grad_weights || (grad_weights & 3) || !grad_logits || (grad_logits & 3)) {
    set_error("asap_route_backward: ids, grad_weights and grad_logits must be non-NULL and 4-byte aligned");
    return ASAP_EINVAL;
  }
  route::BackArgs a{};
  a.logits = (const void*)r->logits;
  a.ld = r->ld;
  a.dtype = r->dtype;
  a.t = r->t;
  a.e = r->e;
  a.k = r->k;
  a.sigmoid = r->sigmoid;
  a.renorm = r->renormalize;
  a.dense = !r->sigmoid && (!r->renormalize || r->bias);
  a.vec = route::rows_16(r->logits, r->ld, r->dtype);
  a.out_vec = route::rows_16(grad_logits, r->e, r->dtype);
  a.scale = r->scale;
  a.ids = (const int32_t*)ids;
  a.grad = (const float*)grad_weights;
  a.out = (void*)grad_logits;
  route::by_experts<route::Backward>(r->e, a, (r->t + route::kWarps - 1) / route::kWarps, (cudaStream_t)stream);
  ASAP_CHECK_LAUNCH("route_back_kernel");
  return ASAP_OK;
}

uint64_t asap_balance_ws_bytes(int32_t t, int32_t seqs) {
  if (t < 1 || t > (1 << 24) || seqs < 1 || seqs > (1 << 20)) return 0;
  return route::balance_ws(t, seqs).bytes;
}

int asap_balance_loss(const asap_balance_t* b, uint64_t ws, uint64_t ws_bytes, uint64_t loss, void* stream) {
  route::BalanceArgs a{};
  if (int rc = route::balance_args("asap_balance_loss", a, b, ws, ws_bytes)) return rc;
  if (!loss || (loss & 3)) {
    set_error("asap_balance_loss: loss must be non-NULL and 4-byte aligned");
    return ASAP_EINVAL;
  }
  a.loss = (float*)loss;
  cudaStream_t st = (cudaStream_t)stream;
  if ((int64_t)b->t * route::per_lane(b->e) <= route::kSmallTokens && (int64_t)b->seqs * b->e <= route::kSmallCounts) {
    route::by_experts<route::LossSmall>(b->e, a, 1, st);
    ASAP_CHECK_LAUNCH("balance_small_kernel");
    return ASAP_OK;
  }
  const uint64_t zeroed = route::balance_ws(b->t, b->seqs).zeroed, cells = 4ull * b->seqs * b->e;
  if (b->counts + cells == ws) {
    ASAP_CUDA(cudaMemsetAsync((void*)b->counts, 0, cells + zeroed, st));
  } else {
    ASAP_CUDA(cudaMemsetAsync((void*)ws, 0, zeroed, st));
    ASAP_CUDA(cudaMemsetAsync((void*)b->counts, 0, cells, st));
  }
  route::balance_count_kernel<<<(b->t + route::kCountRows - 1) / route::kCountRows, route::kCountThreads,
                                4 * (b->e + 1), st>>>(a);
  ASAP_CHECK_LAUNCH("balance_count_kernel");
  route::by_experts<route::Loss>(b->e, a, route::balance_grid(b->t), st);
  ASAP_CHECK_LAUNCH("balance_kernel");
  return ASAP_OK;
}

int asap_balance_backward(const asap_balance_t* b, uint64_t ws, uint64_t ws_bytes, uint64_t grad_loss,
                          uint64_t grad_logits, void* stream) {
  route::BalanceArgs a{};
  if (int rc = route::balance_args("asap_balance_backward", a, b, ws, ws_bytes)) return rc;
  if (!grad_loss || (grad_loss & 3) || !grad_logits || (grad_logits & 3)) {
    set_error("asap_balance_backward: grad_loss and grad_logits must be non-NULL and 4-byte aligned");
    return ASAP_EINVAL;
  }
  a.grad = (const float*)grad_loss;
  a.out = (void*)grad_logits;
  a.out_vec = route::rows_16(grad_logits, b->e, b->dtype);
  route::by_experts<route::LossBack>(b->e, a, route::balance_grid(b->t), (cudaStream_t)stream);
  ASAP_CHECK_LAUNCH("balance_kernel (gradient)");
  return ASAP_OK;
}

int asap_expert_counts(uint64_t ids, int32_t t, int32_t k, int32_t e, uint64_t counts, void* stream) {
  if (!ids || (ids & 3) || !counts || (counts & 3) || t < 1 || t > (1 << 24) || k < 1 || k > ASAP_ROUTE_MAX_TOPK ||
      e < 1 || e > ASAP_ROUTE_MAX_EXPERTS) {
    set_error("asap_expert_counts: need ids and counts (4-byte aligned), 1 to %d tokens, k <= %d, 1 to %d experts (got "
              "%d, %d, %d)", 1 << 24, ASAP_ROUTE_MAX_TOPK, ASAP_ROUTE_MAX_EXPERTS, t, k, e);
    return ASAP_EINVAL;
  }
  route::BalanceArgs a{};
  a.t = t;
  a.e = e;
  a.k = k;
  a.seqs = 1;
  a.ids = (const int32_t*)ids;
  a.counts = (int32_t*)counts;
  cudaStream_t st = (cudaStream_t)stream;
  ASAP_CUDA(cudaMemsetAsync((void*)counts, 0, 4ull * e, st));
  route::balance_count_kernel<<<(t + route::kCountRows - 1) / route::kCountRows, route::kCountThreads,
                                4 * (e + 1), st>>>(a);
  ASAP_CHECK_LAUNCH("balance_count_kernel");
  return ASAP_OK;
}

}  // extern "C"
