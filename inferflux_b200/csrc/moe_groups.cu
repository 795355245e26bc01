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
  int softmax, normalized;
  float floor, scale;
};

constexpr int kGroupRouteMost = 1024;

// Bits ordered as the numbers are; NaN with -inf, and one zero.
__device__ __forceinline__ unsigned long long ordered_bits(double v) {
  if (!(v == v)) v = -INFINITY;
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A warp a token.
__global__ void __launch_bounds__(128) moe_route_groups_kernel(const GroupRouteArgs a) {
  extern __shared__ double v_s[];
  const unsigned all = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * 4 + warp;
  pdl_launch_dependents();
  pdl_wait();
  if (t >= a.T) return;
  double* v = v_s + (size_t)warp * a.n;
  auto logit = [&](int i) {
    float s = a.z[t * a.n + i];
    for (int k = 1; k < a.splits; ++k) s += a.z[(size_t)k * a.split_stride + t * a.n + i];
    return s;
  };
  double m = 0.0, sum = 1.0;
  if (a.softmax) {
    float most = -INFINITY;
    for (int i = lane; i < a.n; i += 32) most = fmaxf(most, logit(i));
    most = warp_max(most);
    m = most == -INFINITY ? 0.0 : (double)most;
    sum = 0.0;
    for (int i = lane; i < a.n; i += 32) sum += exp((double)logit(i) - m);
    sum = warp_sum_f64(sum);
  }
  auto score = [&](int i) {
    const double z = (double)logit(i);
    return a.softmax ? (sum == 0.0 ? 0.0 : exp(z - m) / sum) : 1.0 / (1.0 + exp(-z));
  };
  for (int i = lane; i < a.n; i += 32) v[i] = score(i) + (a.correction ? (double)a.correction[i] : 0.0);
  __syncwarp();
  // a lane a group: its `best` largest, one after the other in falling order
  const int size = a.n / a.groups;
  unsigned long long strength = 0;
  if (lane < a.groups) {
    double total = 0.0;
    unsigned long long before = ~0ull;
    int before_at = -1;
    for (int k = 0; k < a.best; ++k) {
      unsigned long long most = 0;
      int at = -1;
      for (int i = 0; i < size; ++i) {
        const unsigned long long key = ordered_bits(v[lane * size + i]);
        const bool left = key < before || (key == before && i > before_at);
        if (left && (at < 0 || key > most)) { most = key; at = i; }
      }
      total += v[lane * size + at];
      before = most;
      before_at = at;
    }
    strength = ordered_bits(total);
  }
  int place = 0;
  for (int g = 0; g < a.groups; ++g) {
    const unsigned long long other = __shfl_sync(all, strength, g);
    place += other > strength || (other == strength && g < lane);
  }
  const unsigned kept = __ballot_sync(all, lane < a.groups && place < a.kept);
  // the largest of what is left, `top` times; a lane keeps what it has chosen out by one bit an expert of its own
  unsigned taken = 0;
  double mine = 0.0;
  int mine_at = 0;
  for (int c = 0; c < a.top; ++c) {
    unsigned long long most = 0;
    int at = 0x7fffffff;
    for (int i = lane, k = 0; i < a.n; i += 32, ++k) {
      if (taken >> k & 1u || !(kept >> (i / size) & 1u)) continue;
      const unsigned long long key = ordered_bits(v[i]);
      if (at == 0x7fffffff || key > most) { most = key; at = i; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long om = __shfl_xor_sync(all, most, o);
      const int oa = __shfl_xor_sync(all, at, o);
      if (oa != 0x7fffffff && (at == 0x7fffffff || om > most || (om == most && oa < at))) { most = om; at = oa; }
    }
    if ((at & 31) == lane) taken |= 1u << (at >> 5);
    if (lane == c) { mine = score(at); mine_at = at; }
  }
  double total = lane < a.top ? mine : 0.0;
  if (a.normalized) {
    total = warp_sum_f64(total) + (double)a.floor;
    mine = total == 0.0 ? 0.0 : mine / total;
  }
  if (lane < a.top) {
    a.ids[t * a.top + lane] = mine_at;
    a.weights[t * a.top + lane] = (float)(mine * (double)a.scale);
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
  const GroupRouteArgs a{z, splits, (size_t)T * n, correction, ids, weights, T, n, groups, kept, best, top, softmax, normalized, floor, scale};
  return launch_pdl(moe_route_groups_kernel, dim3((unsigned)((T + 3) / 4)), dim3(128), (size_t)4 * n * sizeof(double), stream, 1, a);
}
