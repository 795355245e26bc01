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
  int T, n, groups, kept, best, top;
  int lanes, stride;                                       // lanes of a group, and numbers from one group's first to the next one's in shared memory
  int softmax, normalized;
  float floor, scale;
};

constexpr int kGroupRouteMost = 1024, kGroupRouteWarps = 4;

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

// A warp a token, whose lane has the experts lane, lane + 32, ... (PER of them at most).  Every v goes to shared memory once, group by group; a group's
// lanes find its two largest, and the choice goes through registers: the largest high words by one reduction, the low words and then the
// indices where those are equal.  Bound by the latency of that chain and by the exponentials in float64 (some 25 operations each at half the
// rate of float32).
template <int PER>
__global__ void __launch_bounds__(32 * kGroupRouteWarps) moe_route_groups_kernel(const GroupRouteArgs a) {
  extern __shared__ double v_s[];
  const unsigned all = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kGroupRouteWarps + warp;
  const int size = a.n / a.groups;
  pdl_launch_dependents();
  float correction[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) correction[k] = a.correction && lane + 32 * k < a.n ? a.correction[lane + 32 * k] : 0.0f;
  pdl_wait();
  if (t >= a.T) return;
  double* const mine_s = v_s + (size_t)warp * a.groups * a.stride;
  const float* zr = a.z + t * a.n;
  float z[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) z[k] = lane + 32 * k < a.n ? zr[lane + 32 * k] : -INFINITY;
  for (int s = 1; s < a.splits; ++s)
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (lane + 32 * k < a.n) z[k] += zr[s * a.split_stride + lane + 32 * k];
  double m = 0.0, sum = 1.0;
  if (a.softmax) {
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < PER; ++k) most = fmaxf(most, z[k]);
    most = warp_max(most);
    m = most == -INFINITY ? 0.0 : (double)most;              // (nothing to share out: every exponential is 0)
  }
  auto weight = [&](float zi) { return a.softmax ? exp((double)zi - m) : 1.0 / (1.0 + exp(-(double)zi)); };
  double v[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) v[k] = weight(z[k]);         // (behind the last expert: of -inf, 0)
  if (a.softmax) {
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += v[k];
    sum = warp_sum_f64(sum);
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = sum == 0.0 ? 0.0 : v[k] / sum;
  }
  unsigned short group[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = lane + 32 * k;
    v[k] = number_or_least(v[k] + (double)correction[k]);
    group[k] = (unsigned short)(i / size);
    if (i < a.n && a.groups > 1) mine_s[group[k] * a.stride + i - group[k] * size] = v[k];
  }
  // the groups' strengths, group g's in lane g
  unsigned kept = 1;
  if (a.groups > 1) {
    __syncwarp();
    const int g = lane / a.lanes, sub = lane % a.lanes;
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
    } else {                                                 // one after the other in falling order, by a group's first lane
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
  double w = 0.0;
  if (lane < a.top) {
    float zi = zr[mine_at];
    for (int s = 1; s < a.splits; ++s) zi += zr[s * a.split_stride + mine_at];
    w = weight(zi);
    if (a.softmax) w = sum == 0.0 ? 0.0 : w / sum;
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
  GroupRouteArgs a{z, splits, (size_t)T * n, correction, ids, weights, T, n, groups, kept, best, top, 1, n / groups, softmax, normalized, floor, scale};
  while (2 * a.lanes * groups <= 32) a.lanes *= 2;
  while (a.stride % 16 != a.lanes % 16) ++a.stride;           // a half warp's reads of 8 bytes fall on different banks
  const size_t bytes = (size_t)kGroupRouteWarps * groups * a.stride * sizeof(double);       // 32 groups of 32 experts and one: 34 KB; at most 48
  const dim3 grid((unsigned)((T + kGroupRouteWarps - 1) / kGroupRouteWarps)), block(32 * kGroupRouteWarps);
  auto kernel = n <= 32 ? moe_route_groups_kernel<1> : n <= 64 ? moe_route_groups_kernel<2> : n <= 128 ? moe_route_groups_kernel<4>
              : n <= 256 ? moe_route_groups_kernel<8> : n <= 512 ? moe_route_groups_kernel<16> : moe_route_groups_kernel<32>;
  return launch_pdl(kernel, grid, block, groups > 1 ? bytes : 0, stream, 1, a);
}
