// A state space scan whose decay is made from the input for every channel and every number of its state, and what makes its inputs.
//
//   selective_scan     dt = softplus(raw + bias)
//                      h[c, n] <- exp(-dt e^log_rate[c, n]) h[c, n] + dt x[c] B[n]                 n = 0 .. states - 1
//                      y[c] = (sum_n C[n] h[c, n] + skip[c] x[c]) silu(z[c])
//   selective_inputs   rows [T, rank + 2 states] -> low = the first rank columns in the run's dtype, B | C = the others in float32, each of the
//                      three parts over its own root mean square times a weight (no weight: as it is)
//
// h is float32, [channels, states] per request at `state + slot * slot_stride`; a new request finds it zeroed.  Steps, decays, states and sums
// are float32 whatever the rows' dtype; y is rounded once.
//
// A channel's states are spread over neighbouring lanes, four (or two) a lane.  The sum over n is a tree: neighbouring pairs, pairs of
// pairs, and so on, the same whatever a lane holds, and every h is one chain of multiply-adds from token to token; so a float32 run's
// bits do not depend on how a request's tokens are cut into steps.
#include "common.cuh"

namespace ifx {

struct SelectiveArgs {
  const void* x; long long ld_x; int x_dtype;
  const void* dt; long long ld_dt; int dt_dtype;
  const float* bc; long long ld_bc;
  const void* z; long long ld_z;                   // null: no gate; x's dtype
  const float* log_rate;                           // [channels, states]
  const float* bias;                               // [channels], null: none
  const float* skip;                               // [channels], null: none
  float* state; long long slot_stride;
  const int* req_slot; const int* cu_seqlens;
  void* out; int out_dtype;                        // [T, channels]
  int channels, states;
};

__device__ __forceinline__ float load_as_f32(const void* p, long long at, int dtype) {
  return dtype == IFX_DT_F32 ? static_cast<const float*>(p)[at] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

// log(1 + e^v) = max(v, 0) + log(1 + e^-|v|), and log(1 + e) = 2 artanh(s) with s = e / (2 + e) <= 1/3, by artanh's own series
// s (1 + s^2/3 + s^4/5 + ...): relative to the result, which a logarithm of 1 + e is not where e is small.  The terms left out are below
// (1/9)^8 / 17 = 1.4e-9.
__device__ __forceinline__ float softplus_f32(float v) {
  const float e = exp2_fast(-fabsf(v) * kLog2e);
  const float s = __fdividef(e, 2.0f + e), q = s * s;
  float p = 1.0f / 15.0f;
  p = fmaf(p, q, 1.0f / 13.0f);
  p = fmaf(p, q, 1.0f / 11.0f);
  p = fmaf(p, q, 1.0f / 9.0f);
  p = fmaf(p, q, 1.0f / 7.0f);
  p = fmaf(p, q, 1.0f / 5.0f);
  p = fmaf(p, q, 1.0f / 3.0f);
  p = fmaf(p, q, 1.0f);
  return fmaf(2.0f * s, p, fmaxf(v, 0.0f));
}

__device__ __forceinline__ float silu_f32(float z) {
  const float e = exp2_fast(-fabsf(z) * kLog2e);                   // the divisor lies between 1 and 2
  const float big = __fdividef(1.0f, 1.0f + e);
  return z * (z >= 0.0f ? big : e * big);
}

// A token of one lane's states: the step's decay and input go into h, and the lane's part of the sum over n comes back.  `real`: how many of
// the lane's states there are; the others stay 0 (an infinite x times their zero B would be NaN).
template <int S, bool PAD>
__device__ __forceinline__ float selective_token(float (&h)[S], const float (&rate2)[S], float dt, float dtx, const float (&b)[S],
                                                 const float (&c)[S], int real) {
#pragma unroll
  for (int j = 0; j < S; ++j) {
    h[j] = fmaf(exp2_fast(dt * rate2[j]), h[j], dtx * b[j]);
    if (PAD && j >= real) h[j] = 0.0f;
  }
  float y = fmaf(c[1], h[1], c[0] * h[0]);
#pragma unroll
  for (int j = 2; j < S; j += 2) y += fmaf(c[j + 1], h[j + 1], c[j] * h[j]);
  return y;
}

// LANES lanes a channel, four states a lane; a block of 128 threads walks one request's tokens.
template <int LANES, bool PAD>
__global__ void __launch_bounds__(128) selective_scan_kernel(const SelectiveArgs a) {
  constexpr int S = 4;
  const int c = (blockIdx.x * 128 + threadIdx.x) / LANES, part = threadIdx.x % LANES, n0 = part * S, r = blockIdx.y;
  const bool live = c < a.channels;
  pdl_launch_dependents();
  const long long first = a.cu_seqlens[r], last = a.cu_seqlens[r + 1];
  float* st = a.state + (long long)a.req_slot[r] * a.slot_stride + (long long)c * a.states + n0;
  float rate2[S], h[S], b[S], cc[S];
#pragma unroll
  for (int j = 0; j < S; ++j) rate2[j] = live && n0 + j < a.states ? -expf(a.log_rate[(long long)c * a.states + n0 + j]) * kLog2e : 0.0f;
  const float bias = live && a.bias ? a.bias[c] : 0.0f, skip = live && a.skip ? a.skip[c] : 0.0f;
  pdl_wait();
  if (first >= last) return;
#pragma unroll
  for (int j = 0; j < S; ++j) h[j] = live && n0 + j < a.states ? st[j] : 0.0f;
  for (long long t = first; t < last; ++t) {
    const float x = live ? load_as_f32(a.x, t * a.ld_x + c, a.x_dtype) : 0.0f;
    const float dt = live ? softplus_f32(load_as_f32(a.dt, t * a.ld_dt + c, a.dt_dtype) + bias) : 0.0f;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      b[j] = n0 + j < a.states ? a.bc[t * a.ld_bc + n0 + j] : 0.0f;
      cc[j] = n0 + j < a.states ? a.bc[t * a.ld_bc + a.states + n0 + j] : 0.0f;
    }
    float y = selective_token<S, PAD>(h, rate2, dt, dt * x, b, cc, a.states - n0);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (live && part == 0) {
      if (a.skip) y = fmaf(skip, x, y);                       // (no skip is not one of zero: x may be infinite)
      if (a.z) y *= silu_f32(load_as_f32(a.z, t * a.ld_z + c, a.x_dtype));
      const long long at = t * a.channels + c;
      if (a.out_dtype == IFX_DT_F32) static_cast<float*>(a.out)[at] = y;
      else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y);
    }
  }
#pragma unroll
  for (int j = 0; j < S; ++j)
    if (live && n0 + j < a.states) st[j] = h[j];
}

struct SelectiveInputsArgs {
  const void* rows; long long ld; int dtype, splits; size_t split_stride;
  const float* w_low; const float* w_b; const float* w_c;      // null: that part is not normed
  float eps;
  void* low; int low_dtype;
  float* bc;
  int T, rank, states;
};

// A warp a row, which it keeps in shared memory between the sum of squares and the result.
__global__ void __launch_bounds__(128) selective_inputs_kernel(const SelectiveInputsArgs a) {
  extern __shared__ float rows_s[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, width = a.rank + 2 * a.states;
  const long long t = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  pdl_launch_dependents();
  pdl_wait();
  if (t >= a.T) return;
  float* row = rows_s + (size_t)warp * width;
  for (int part = 0; part < 3; ++part) {
    const int col0 = part == 0 ? 0 : a.rank + (part - 1) * a.states, n = part == 0 ? a.rank : a.states;
    const float* w = part == 0 ? a.w_low : part == 1 ? a.w_b : a.w_c;
    float ss = 0.0f;
    for (int i = lane; i < n; i += 32) {
      const long long at = t * a.ld + col0 + i;
      float v = load_as_f32(a.rows, at, a.dtype);
      for (int s = 1; s < a.splits; ++s) v += static_cast<const float*>(a.rows)[(size_t)s * a.split_stride + at];
      row[col0 + i] = v;
      ss = fmaf(v, v, ss);
    }
    const float scale = w ? rsqrtf(warp_sum(ss) / (float)n + a.eps) : 1.0f;
    for (int i = lane; i < n; i += 32) {
      const float v = w ? row[col0 + i] * scale * w[i] : row[col0 + i];
      if (part) a.bc[t * 2 * a.states + (part - 1) * a.states + i] = v;
      else if (a.low_dtype == IFX_DT_F32) static_cast<float*>(a.low)[t * a.rank + i] = v;
      else static_cast<__nv_bfloat16*>(a.low)[t * a.rank + i] = __float2bfloat16_rn(v);
    }
  }
}

}  // namespace ifx

using namespace ifx;

static bool known_dtype(int d) { return d == IFX_DT_F32 || d == IFX_DT_BF16; }

// Row strides in elements.  x and z share a dtype; bc: float32 rows of B | C; state: float32, slots slot_stride floats apart.
// num_tokens: rows of x; cu_seqlens does not go beyond them.  A request without tokens keeps its state.
extern "C" int ifx_selective_scan(const void* x, long long ld_x, int x_dtype, const void* dt, long long ld_dt, int dt_dtype, const float* bc,
                                  long long ld_bc, const void* z, long long ld_z, const float* log_rate, const float* bias, const float* skip,
                                  float* state, long long slot_stride, const int* req_slot, const int* cu_seqlens, void* out, int out_dtype,
                                  int num_requests, int num_tokens, int max_span, int channels, int states, cudaStream_t stream) {
  if (num_requests < 0 || num_tokens < 0 || max_span < 0 || channels <= 0 || states <= 0) return IFX_E_BADARG;
  if (!known_dtype(x_dtype) || !known_dtype(dt_dtype) || !known_dtype(out_dtype)) return IFX_E_DTYPE;
  if (states > 128 || num_requests > 65535) return IFX_E_TOOBIG;
  if (num_requests == 0 || num_tokens == 0 || max_span == 0) return 0;
  if (ld_x < channels || ld_dt < channels || (z && ld_z < channels) || ld_bc < 2 * states || slot_stride < (long long)channels * states)
    return IFX_E_BADARG;
  if (!x || !dt || !bc || !log_rate || !state || !req_slot || !cu_seqlens || !out) return IFX_E_BADARG;
  const SelectiveArgs a{x, ld_x, x_dtype, dt, ld_dt, dt_dtype, bc, ld_bc, z, ld_z, log_rate, bias, skip, state, slot_stride, req_slot, cu_seqlens,
                        out, out_dtype, channels, states};
  int lanes = 1;
  while (lanes * 4 < states) lanes <<= 1;
  const dim3 grid((unsigned)(((long long)channels * lanes + 127) / 128), num_requests);
  const bool pad = states != lanes * 4;
#define IFX_SELECTIVE(L) case L: return launch_pdl(pad ? selective_scan_kernel<L, true> : selective_scan_kernel<L, false>, grid, dim3(128), 0, stream, 1, a)
  switch (lanes) {
    IFX_SELECTIVE(1); IFX_SELECTIVE(2); IFX_SELECTIVE(4); IFX_SELECTIVE(8); IFX_SELECTIVE(16);
    IFX_SELECTIVE(32);
  }
  return IFX_E_BADARG;
#undef IFX_SELECTIVE
}

// rows: [T, rank + 2 states], ld elements apart; splits > 1: float32, the partial sums [splits, T, rank + 2 states] of a K-split product.
// low: [T, rank]; bc: float32 [T, 2 states].
extern "C" int ifx_selective_inputs(const void* rows, long long ld, int dtype, int splits, const float* w_low, const float* w_b, const float* w_c,
                                    float eps, void* low, int low_dtype, float* bc, int T, int rank, int states, cudaStream_t stream) {
  if (T < 0 || rank <= 0 || states <= 0 || splits < 1 || ld < (long long)rank + 2 * states) return IFX_E_BADARG;
  if (!known_dtype(dtype) || !known_dtype(low_dtype) || (splits > 1 && dtype != IFX_DT_F32)) return IFX_E_DTYPE;
  if (rank > 8192 || states > 1024) return IFX_E_TOOBIG;
  if (T == 0) return 0;
  if (!rows || !low || !bc) return IFX_E_BADARG;
  const SelectiveInputsArgs a{rows, ld, dtype, splits, (size_t)T * ld, w_low, w_b, w_c, eps, low, low_dtype, bc, T, rank, states};
  const int width = rank + 2 * states;
  const int warps = width <= 3000 ? 4 : 1;                       // of at most 48 KB of rows a block
  return launch_pdl(selective_inputs_kernel, dim3((unsigned)((T + warps - 1) / warps)), dim3(32 * warps), (size_t)warps * width * 4, stream, 1, a);
}
