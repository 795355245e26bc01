// A router's choice with experts in groups: only the experts of a token's best groups are chosen from.
//
//   s = sigmoid(z) or softmax(z) over all experts,   v = s + correction
//   a group's strength = the sum of the `best` largest v of its experts;   the `kept` groups of the greatest strength stay
//   ids = the `top` experts of those groups with the largest v, falling;   weights = s[ids] (over (their sum + floor)) * scale
//
// Ties go to the lower index, of groups and of experts.  Which of two near numbers is the larger is decided in float64: a choice must not
// depend on how float32 rounds an exponential.  Every row gets `top` different experts of its kept groups whatever its logits are: a v that is
// not a number counts as -inf, and a row whose softmax has nothing to share out (all -inf) has scores of zero.
#include "common.cuh"

namespace ifx {

struct GroupRouteArgs {
  const float* z; int splits; size_t split_stride;         // [splits, T, n] partial sums, added in split order
  const float* correction;                                 // [n] or null
  int* ids; float* weights;                                // [T, top]
  int T, n, groups, size, kept, best, top;                 // size: experts of a group
  int lanes, lane_bits, stride;                            // lanes of a group (a power of two), and numbers from one group's first to the next one's
  unsigned by_size;                                        // in shared memory; expert i is in group i by_size >> 20 (exact: i, n / groups <= 2^10)
  int softmax, normalized;
  float floor, scale;
};

constexpr int kGroupRouteMost = 1024, kGroupRouteWarps = 2;

// Bits ordered as the numbers are, of numbers alone (one zero); 0 stands before all of them.
__device__ __forceinline__ unsigned long long ordered_bits(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double number_or_least(double v) { return v == v ? v : -INFINITY; }

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ unsigned ordered_bits(float v) {
  const unsigned u = __float_as_uint(v + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// Logit i of the token whose first lies at `zr`: slices are added in their order.
__device__ __forceinline__ float logit(const GroupRouteArgs& a, const float* zr, int i) {
  float z = zr[i];
  for (int s = 1; s < a.splits; ++s) z += zr[s * a.split_stride + i];
  return z;
}

// (one copy for all its callers: the rare ones find it in the instruction cache)
__device__ __noinline__ double exact_score(const GroupRouteArgs& a, float z, float m, double sum) {
  return !a.softmax ? 1.0 / (1.0 + exp(-(double)z)) : sum == 0.0 ? 0.0 : exp((double)z - (double)m) / sum;
}

// One token by a warp.  zr: its logits.  Both give the choice, number c in lane c.
//
// In float64, where a lane has the experts lane, lane + 32, ... (PER of them at most): every v goes to shared memory, group by group; a group's lanes find its two largest (more: its first lane does, one after the
// other), and the choice goes through registers: the largest high words by one reduction, the low words and then the indices where those are
// equal.
template <int PER>
__device__ __noinline__ int choose_exactly(const GroupRouteArgs& a, const float* zr, double* mine_s) {
  const unsigned all = 0xffffffffu;
  const int lane = threadIdx.x & 31, size = a.size;
  float z[PER];
  unsigned char group[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = lane + 32 * k;
    z[k] = i < a.n ? logit(a, zr, i) : -INFINITY;
    group[k] = (unsigned char)(i * a.by_size >> 20);
  }
  double m = 0.0, sum = 1.0;
  if (a.softmax) {
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; ++k) most = fmaxf(most, z[k]);
    most = warp_max(most);
    m = most == -INFINITY ? 0.0 : (double)most;              // (nothing to share out: every exponential is 0)
  }
  double v[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) v[k] = a.softmax ? exp((double)z[k] - m) : 1.0 / (1.0 + exp(-(double)z[k]));     // (behind the last expert 0)
  if (a.softmax) {
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += v[k];
    sum = warp_sum_f64(sum);
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = sum == 0.0 ? 0.0 : v[k] / sum;
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = lane + 32 * k;
    v[k] = number_or_least(v[k] + (a.correction && i < a.n ? (double)a.correction[i] : 0.0));
    if (i < a.n && a.groups > 1) mine_s[group[k] * a.stride + i - group[k] * size] = v[k];
  }
  // the groups' strengths, group g's in lane g
  unsigned kept = 1;
  if (a.groups > 1) {
    __syncwarp();
    const int g = lane >> a.lane_bits, sub = lane & (a.lanes - 1);
    const double* members = mine_s + min(g, a.groups - 1) * a.stride;
    double strength;
    if (a.best <= 2) {
      double first = -INFINITY, second = -INFINITY;
      for (int i = sub; i < size; i += a.lanes) {
        const double w = members[i];
        second = fmax(second, fmin(first, w));
        first = fmax(first, w);
      }
      for (int o = 1; o < a.lanes; o <<= 1) {
        const double other = __shfl_xor_sync(all, first, o), next = __shfl_xor_sync(all, second, o);
        second = fmax(fmin(first, other), fmax(second, next));
        first = fmax(first, other);
      }
      strength = a.best == 1 ? first : first + second;
    } else {
      strength = 0.0;
      unsigned long long before = ~0ull;
      int before_at = -1;
      for (int c = 0; c < a.best && sub == 0; ++c) {
        unsigned long long largest = 0;
        int at = 0;
        for (int i = 0; i < size; ++i) {
          const unsigned long long key = ordered_bits(members[i]);
          if ((key < before || (key == before && i > before_at)) && key > largest) { largest = key; at = i; }
        }
        strength += members[at];
        before = largest;
        before_at = at;
      }
    }
    __syncwarp();
    strength = __shfl_sync(all, number_or_least(strength), min(lane, a.groups - 1) * a.lanes);
    int place = 0;
    for (int j = 0; j < a.groups; ++j) {
      const double other = __shfl_sync(all, strength, j);
      place += other > strength || (other == strength && j < lane);
    }
    kept = __ballot_sync(all, lane < a.groups && place < a.kept);
  }
  // the choice: a lane's candidates as ordered bits (0: none), the best of them first
  unsigned hi[PER], lo[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const bool in = lane + 32 * k < a.n && (kept >> group[k] & 1u);
    const unsigned long long key = in ? ordered_bits(v[k]) : 0ull;
    hi[k] = (unsigned)(key >> 32);
    lo[k] = (unsigned)key;
  }
  unsigned best_hi = 0, best_lo = 0;
  int best_k = 0;
  auto find = [&]() {
    best_hi = best_lo = 0;
    best_k = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (hi[k] > best_hi || (hi[k] == best_hi && lo[k] > best_lo)) { best_hi = hi[k]; best_lo = lo[k]; best_k = k; }
  };
  find();
  int mine_at = 0;
  for (int c = 0; c < a.top; ++c) {
    const unsigned most = __reduce_max_sync(all, best_hi);
    unsigned who = __ballot_sync(all, best_hi == most);
    if (who & (who - 1)) {                                   // several with this high word
      const unsigned low = __reduce_max_sync(all, best_hi == most ? best_lo : 0u);
      const bool in = best_hi == most && best_lo == low;
      const unsigned least = __reduce_min_sync(all, in ? (unsigned)(lane + 32 * best_k) : 0xffffffffu);
      who = __ballot_sync(all, in && lane + 32 * best_k == (int)least);
    }
    const int winner = __ffs(who) - 1, at = __shfl_sync(all, lane + 32 * best_k, winner);
    if (lane == c) mine_at = at;
    if (lane == winner) {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (k == best_k) hi[k] = lo[k] = 0;
      find();
    }
  }
  return mine_at;
}

// Where a lane's experts are in choose_fast: `lanes` lanes have a group, so that its strength takes registers alone.
struct GroupLane {
  int first, count, bits;                                    // its k-th of `count` is expert first + (k << bits)
  __device__ __forceinline__ explicit GroupLane(const GroupRouteArgs& a) : bits(a.lane_bits) {
    const int lane = threadIdx.x & 31, g = lane >> a.lane_bits, sub = lane & (a.lanes - 1);
    first = g * a.size + sub;
    count = g < a.groups ? (a.size - sub + a.lanes - 1) >> a.lane_bits : 0;
  }
  __device__ __forceinline__ int at(int k) const { return first + (k << bits); }
};

// The same in float32, in which experts and groups that are nearer than their errors are told apart in float64 on the spot.  False, and nothing
// said, where three experts of one lane are that near, more of a group than its strength counts, or where a number is none.
// v: -inf behind the lane's last.
//
// A score is off by less than 2^-21: a sigmoid by (0.76 + 0.5 + 2) 2^-23, of which the fast exponential of x, good to 2 + 1.173 |x| steps, makes
// s (1 - s) (2 + 1.173 |x|) <= 0.76 of them, the sum half a one, and the fast quotient two; a softmax's, by three roundings of what float64 gave.  v is off
// by half a step of its own more, a strength by its terms' errors and a rounding a sum.
template <int PER>
__device__ __forceinline__ bool choose_fast(const GroupRouteArgs& a, const float* zr, float m, double sum, const float (&v)[PER],
                                            const GroupLane& own, int& chosen) {
  const unsigned all = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  bool in_kept = true;
  if (a.groups > 1) {
    if (a.best > 4) return false;
    float strength, magnitude, least_term = 0.0f;            // of its terms
    bool numbers = true;                                     // (the largest of a NaN and a number is the number)
#pragma unroll
    for (int k = 0; k < PER; ++k) numbers = numbers && v[k] == v[k];
    if (!__all_sync(all, numbers)) return false;
    if (a.best <= 2) {
      float first = -INFINITY, next = -INFINITY;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        next = fmaxf(next, fminf(first, v[k]));
        first = fmaxf(first, v[k]);
      }
      for (int o = 1; o < a.lanes; o <<= 1) {
        const float other = __shfl_xor_sync(all, first, o);
        next = fmaxf(fminf(first, other), fmaxf(next, __shfl_xor_sync(all, next, o)));
        first = fmaxf(first, other);
      }
      strength = a.best == 1 ? first : first + next;
      magnitude = fabsf(first) + (a.best == 1 ? 0.0f : fabsf(next));
      least_term = a.best == 1 ? first : next;
    } else {
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      auto insert = [&](float w) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float less = fminf(top[j], w);
          top[j] = fmaxf(top[j], w);
          w = less;
        }
      };
#pragma unroll
      for (int k = 0; k < PER; ++k) insert(v[k]);
      for (int o = 1; o < a.lanes; o <<= 1) {
        float other[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) other[j] = __shfl_xor_sync(all, top[j], o);
#pragma unroll
        for (int j = 0; j < 4; ++j) insert(other[j]);
      }
      strength = top[0] + top[1] + top[2] + (a.best == 4 ? top[3] : 0.0f);
      magnitude = fabsf(top[0]) + fabsf(top[1]) + fabsf(top[2]) + (a.best == 4 ? fabsf(top[3]) : 0.0f);
    }
    const bool real = lane >> a.lane_bits < a.groups;        // (lanes behind the last group have none)
    int place = 0;
    for (int j = 0; j < a.groups; ++j) place += __shfl_sync(all, strength, j << a.lane_bits) > strength;
    in_kept = real && place < a.kept;
    if (a.kept < a.groups) {
      const int kept = __popc(__ballot_sync(all, in_kept));
      const float inside = from_ordered(__reduce_min_sync(all, in_kept ? ordered_bits(strength) : 0xffffffffu));
      const float outside = from_ordered(__reduce_max_sync(all, real && !in_kept ? ordered_bits(strength) : 0u));
      const float most = __uint_as_float(__reduce_max_sync(all, real ? __float_as_uint(magnitude) : 0u));
      const float error = 0x1p-20f + most * 0x1p-20f;        // of two terms; of two strengths so many times as they have terms, and one for their sums
      if (!(most < INFINITY)) return false;
      if (kept != a.kept << a.lane_bits || !(inside - outside > (a.best + 1) * error)) {
        // every group's strength from its largest terms in float64, if those are clear
        if (a.best > 2) return false;
        unsigned long long counts = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (k < own.count && v[k] >= least_term - error) counts |= 1ull << k;
        double exact = 0.0;
        int terms = __popcll(counts);
        while (__any_sync(all, counts != 0)) {
          if (counts) {
            const int i = own.at(__ffsll(counts) - 1);
            exact += exact_score(a, logit(a, zr, i), m, sum) + (a.correction ? (double)a.correction[i] : 0.0);
            counts &= counts - 1;
          }
          __syncwarp();
        }
        for (int o = 1; o < a.lanes; o <<= 1) {              // (two terms' sum: in either order)
          exact += __shfl_xor_sync(all, exact, o);
          terms += __shfl_xor_sync(all, terms, o);
        }
        if (!__all_sync(all, !real || terms == a.best)) return false;
        place = 0;
        for (int j = 0; j < a.groups; ++j) {
          const double other = __shfl_sync(all, exact, j << a.lane_bits);
          place += other > exact || (other == exact && j < lane >> a.lane_bits);
        }
        in_kept = real && place < a.kept;
      }
    }
  }
  // a lane's candidates (0: none) in falling order, each with its number k in the low bits, which the order's last bits give way to
  constexpr unsigned kLow = PER - 1;
  unsigned key[PER];
  const int candidates = in_kept ? own.count : 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) key[k] = k < candidates ? (ordered_bits(v[k]) & ~kLow) | (unsigned)k : 0u;
#pragma unroll
  for (int length = 2; length <= PER; length *= 2)           // bitonic merges
#pragma unroll
    for (int apart_by = length / 2; apart_by > 0; apart_by /= 2)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int j = apart_by == length / 2 ? i ^ (length - 1) : i ^ apart_by;      // (the first of a merge: mirrored)
        if (j > i) {
          const unsigned large = max(key[i], key[j]);
          key[j] = min(key[i], key[j]);
          key[i] = large;
        }
      }
  for (int c = 0; c < a.top; ++c) {
    const float value = from_ordered(__reduce_max_sync(all, key[0]) & ~kLow);
    if (!(value - value == 0.0f)) return false;              // no number
    // those that may be the largest: one alone, or told apart in float64, of a lane's first two at most
    const unsigned near = ordered_bits(value - (0x1p-20f + fabsf(value) * (0x1p-20f + PER * 0x1p-22f)));
    const bool in = key[0] >= near;                          // (truncated keys on one side only: their last bits are in the bound)
    unsigned who = __ballot_sync(all, in);
    const bool two = PER > 1 && key[PER > 1 ? 1 : 0] >= near;
    if ((who & (who - 1)) || (PER > 1 && __any_sync(all, two))) {
      if (PER > 2 && __any_sync(all, key[PER > 2 ? 2 : 0] >= near)) return false;
      double most = -INFINITY;
      int at = 0x7fffffff;
#pragma unroll 1
      for (int j = 0; j < (PER > 1 ? 2 : 1); ++j) {
        const int i = own.at((int)(key[PER > 1 && j ? 1 : 0] & kLow));
        if (j ? two : in) {
          const double other = exact_score(a, logit(a, zr, i), m, sum) + (a.correction ? (double)a.correction[i] : 0.0);
          if (other > most || (other == most && i < at)) {
            if (j) {                                         // the second is the first
              const unsigned swap = key[0];
              key[0] = key[PER > 1 ? 1 : 0];
              key[PER > 1 ? 1 : 0] = swap;
            }
            most = other;
            at = i;
          }
        }
      }
      const int mine = at;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double other = __shfl_xor_sync(all, most, o);
        const int other_at = __shfl_xor_sync(all, at, o);
        if (other > most || (other == most && other_at < at)) { most = other; at = other_at; }
      }
      who = __ballot_sync(all, in && mine == at);
    }
    const int winner = __ffs(who) - 1, at = __shfl_sync(all, own.at((int)(key[0] & kLow)), winner);
    if (lane == c) chosen = at;
    if (lane == winner) {
#pragma unroll
      for (int k = 0; k + 1 < PER; ++k) key[k] = key[k + 1];
      key[PER - 1] = 0;
    }
  }
  return true;
}

// A warp a token.  Bound by the latency of one token's chain (a decode batch) and by the instructions of all (prompts).  A lane's experts are
// all of one group, so that strengths take registers and `lanes` - 1 shuffles, not a row in shared memory (us, 8,192 tokens of 256 experts in 8
// groups 15.1 for 16.6, 2,047 of 160 5.9 / 6.8, 24 of 256 3.7 / 4.0).  Two warps a block, four, eight: 14.8, 15.1, 15.9; 24 tokens 3.5, 3.7, 4.1.
// Without the choice's rounds but the first 11.4, without the groups 13.6, with weights in float32 13.7.
template <int PER>
__global__ void __launch_bounds__(32 * kGroupRouteWarps) moe_route_groups_kernel(const GroupRouteArgs a) {
  extern __shared__ double v_s[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kGroupRouteWarps + warp;
  pdl_launch_dependents();
  const GroupLane own(a);
  float correction[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) correction[k] = a.correction && k < own.count ? a.correction[own.at(k)] : 0.0f;
  pdl_wait();
  if (t >= a.T) return;
  const float* zr = a.z + t * a.n;
  float z[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) z[k] = k < own.count ? zr[own.at(k)] : -INFINITY;
  for (int s = 1; s < a.splits; ++s)
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (k < own.count) z[k] += zr[s * a.split_stride + own.at(k)];
  float score[PER], m = 0.0f;
  double sum = 1.0;                                          // (in float64: every weight is rounded once)
  if (a.softmax) {
    m = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; ++k) m = fmaxf(m, z[k]);
    m = warp_max(m);
    m = m == -INFINITY ? 0.0f : m;                           // (nothing to share out: every exponential is 0)
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const double e = exp((double)z[k] - (double)m);
      sum += e;
      score[k] = (float)e;
    }
    sum = warp_sum_f64(sum);
    const float share = sum == 0.0 ? 0.0f : (float)(1.0 / sum);
#pragma unroll
    for (int k = 0; k < PER; ++k) score[k] *= share;
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) {                          // (__fdividef: divisors below 2^126)
      const float s = __fdividef(1.0f, 1.0f + __expf(fminf(-z[k], 80.0f)));
      score[k] = z[k] == z[k] ? s : z[k];
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) score[k] = k < own.count ? score[k] + correction[k] : -INFINITY;
  int mine_at = 0;
  if (!choose_fast<PER>(a, zr, m, sum, score, own, mine_at)) {
    __syncwarp();
    mine_at = choose_exactly<PER < 32 ? PER : 32>(a, zr, v_s + (size_t)warp * a.groups * a.stride);      // (32 PER >= n)
  }
  double w = 0.0;
  if (lane < a.top) {
    w = exact_score(a, logit(a, zr, mine_at), m, sum);
  }
  if (a.normalized) {
    const double total = warp_sum_f64(w) + (double)a.floor;
    w = total == 0.0 ? 0.0 : w / total;
  }
  if (lane < a.top) {
    a.ids[t * a.top + lane] = mine_at;
    a.weights[t * a.top + lane] = (float)(w * (double)a.scale);
  }
}

}  // namespace ifx

using namespace ifx;

// z: float32 [splits, T, n] (splits 1: plain).
extern "C" int ifx_moe_route_groups(const float* z, int splits, const float* correction, int* ids, float* weights, int T, int n, int groups,
                                    int kept, int best, int top, int softmax, int normalized, float floor, float scale, cudaStream_t stream) {
  if (T < 0 || splits < 1 || n <= 0 || groups <= 0 || n % groups || kept < 1 || kept > groups || best < 1 || best > n / groups || top < 1 ||
      top > kept * (n / groups))
    return IFX_E_BADARG;
  if (n > kGroupRouteMost || groups > 32 || top > 32) return IFX_E_TOOBIG;
  if (T == 0) return 0;
  if (!z || !ids || !weights) return IFX_E_BADARG;
  const int size = n / groups;
  GroupRouteArgs a{z, splits, (size_t)T * n, correction, ids, weights, T, n, groups, size, kept, best, top, 1, 0, size,
                   ((1u << 20) + size - 1) / size, softmax, normalized, floor, scale};
  while (2 * a.lanes * groups <= 32) {
    a.lanes *= 2;
    ++a.lane_bits;
  }
  while (a.stride % 16 != a.lanes % 16) ++a.stride;           // a half warp's reads of 8 bytes fall on different banks
  const size_t bytes = (size_t)kGroupRouteWarps * groups * a.stride * sizeof(double);       // 32 groups of 32 experts and one: 17 KB; at most 24
  const dim3 grid((unsigned)((T + kGroupRouteWarps - 1) / kGroupRouteWarps)), block(32 * kGroupRouteWarps);
  const int per = (size + a.lanes - 1) / a.lanes;             // of a lane: up to 60, as 17 groups of 60 have a lane each
  auto kernel = per <= 1 ? moe_route_groups_kernel<1> : per <= 2 ? moe_route_groups_kernel<2> : per <= 4 ? moe_route_groups_kernel<4>
              : per <= 8 ? moe_route_groups_kernel<8> : per <= 16 ? moe_route_groups_kernel<16> : per <= 32 ? moe_route_groups_kernel<32>
                                                                                                          : moe_route_groups_kernel<64>;
  return launch_pdl(kernel, grid, block, groups > 1 ? bytes : 0, stream, 1, a);
}
