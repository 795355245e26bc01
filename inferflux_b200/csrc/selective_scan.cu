// A state space scan whose decay is made from the input for every channel and every number of its state, and what makes its inputs.
//
//   selective_scan     dt = softplus(raw + bias)
//                      h[c, n] <- exp(-dt e^log_rate[c, n]) h[c, n] + dt x[c] B[n]                 n = 0 .. states - 1
//                      y[c] = (sum_n C[n] h[c, n] + skip[c] x[c]) silu(z[c])
//   selective_inputs   rows [T, rank + 2 states] -> low = the first rank columns in the run's dtype, B | C = the others in float32, each of the
//                      three parts over its own root mean square times a weight (no weight: as it is)
//
// h is float32, [channels, states] per request at `state + slot * slot_stride`; a new request finds it zeroed.  Steps, decays, states and sums
// are float32 whatever the rows' dtype; y is rounded once.  Steps and gates are good to a float32 step or two (measured: 3.6e-7, 3.2e-7 at most).
// Decays are the exponential unit's, good to two: there is one for every token, channel and state number, and they are what a scan's time goes to
// (three float32 prompts of 700 tokens, against 64 bits: 5.0e-7, the plain form 3.0e-7; with decays rounded correctly 1.1e-7, and seven times as long).
//
// A channel's states are spread over lanes, four a lane.  A lane adds its terms as (0 and 2) and (1 and 3), the lanes' sums are added as a tree,
// neighbours first, and every h is one chain of multiply-adds from token to token, whichever kernel walks; so a float32 run's bits do not depend
// on how a request's tokens are cut into steps.
#include <cfloat>
#include <type_traits>

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
  int per_block;                                   // channels of a block of the span kernel
  int stretch, pass; float* ends;                  // spans by stretches: see there (pass 0: whole)
  int wide;                                        // by 16 bytes (8 for bfloat16 rows): 1 x, 2 dt, 4 z, 8 bc, 16 out, 32 state, 64 log_rate
};

__device__ __forceinline__ float load_as_f32(const void* p, long long at, int dtype) {
  return dtype == IFX_DT_F32 ? static_cast<const float*>(p)[at] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}

// The same in two steps, so that several reads are under way before the first is looked at.
__device__ __forceinline__ uint32_t load_raw(const void* p, long long at, int dtype) {
  return dtype == IFX_DT_F32 ? static_cast<const uint32_t*>(p)[at] : static_cast<const unsigned short*>(p)[at];
}
__device__ __forceinline__ float raw_f32(uint32_t raw, int dtype) { return __uint_as_float(dtype == IFX_DT_F32 ? raw : raw << 16); }

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float rcp_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// e^-min(|v|, 104), which is 0 from 87.4 on.  |v| log2 e is rounded to a float32 before the exponential sees it, which alone would make the result off
// by up to |v| 2^-24; what the rounding and log2 e's own left out is added behind it.  (The limit keeps infinities out of the differences; a v that
// is no number stays none.)
__device__ __forceinline__ float exp_minus_abs(float v) {
  constexpr float kLog2eRest = 1.925963033500e-8f, kLn2 = 0.6931471805599453f;       // log2 e - kLog2e
  float a;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(fabsf(v)), "f"(104.0f));
  const float t = -a * kLog2e, rest = fmaf(-a, kLog2eRest, fmaf(-a, kLog2e, -t)), e = exp2_fast(t);
  return fmaf(e, rest * kLn2, e);
}

// log(1 + e^v) = max(v, 0) + log(1 + e^-|v|), and log(1 + e) = 2 artanh(s) with s = e / (2 + e) <= 1/3: relative to the result, which a
// logarithm of 1 + e is not where e is small.  2 artanh(s) / s as the polynomial of degree four in s^2 whose largest relative error on
// [0, 1/9] is the least (by Remez' exchange; 8e-9 with its coefficients rounded to float32).
__device__ __forceinline__ float softplus_f32(float v) {
  const float e = exp_minus_abs(v);
  const float s = e * rcp_fast(2.0f + e), q = s * s;
  float p = 0.2817833423614502f;
  p = fmaf(p, q, 0.27960601449012756f);
  p = fmaf(p, q, 0.40024909377098083f);
  p = fmaf(p, q, 0.6666631698608398f);
  p = fmaf(p, q, 2.0f);
  return fmaf(s, p, fmaxf(v, 0.0f));
}

// z / (1 + e^-z) = z e^min(z, 0) / (1 + e^-|z|); its limit 0 below -87.4
__device__ __forceinline__ float silu_f32(float z) {
  const float e = exp_minus_abs(z);
  return z * ((z < 0.0f ? e : 1.0f) * rcp_fast(1.0f + e));
}

// Two numbers at once: each half is rounded as the scalar operation rounds it.
__device__ __forceinline__ float2 mul_f32x2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma_f32x2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(r))
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return r;
}

// The states of one lane, in pairs.
template <int S>
struct LaneStates {
  float2 v[S / 2];
  __device__ __forceinline__ void load(const float* p, int real) {
#pragma unroll
    for (int j = 0; j < S / 2; ++j) v[j] = make_float2(2 * j < real ? p[2 * j] : 0.0f, 2 * j + 1 < real ? p[2 * j + 1] : 0.0f);
  }
  __device__ __forceinline__ void load_wide(const float* p) {
    if constexpr (S == 4) {
      const float4 f = *reinterpret_cast<const float4*>(p);
      v[0] = make_float2(f.x, f.y);
      v[1] = make_float2(f.z, f.w);
    } else {
      v[0] = *reinterpret_cast<const float2*>(p);
    }
  }
  __device__ __forceinline__ void store(float* p, int real) const {
#pragma unroll
    for (int j = 0; j < S / 2; ++j) {
      if (2 * j < real) p[2 * j] = v[j].x;
      if (2 * j + 1 < real) p[2 * j + 1] = v[j].y;
    }
  }
  __device__ __forceinline__ void store_wide(float* p) const {
    if constexpr (S == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    else *reinterpret_cast<float2*>(p) = v[0];
  }
  // log_rate in, -e^log_rate log2 e out, float32's lowest number where that is beyond it: any step of 2^-119 and more makes a decay of 0 of it, and a
  // step of 0 one of 1, not 0 * -inf.  (A rate that is no number stays none.)
  __device__ __forceinline__ static float rate2_of(float log_rate) {
    const float r = -expf(log_rate) * kLog2e;
    return r < -FLT_MAX ? -FLT_MAX : r;
  }
  __device__ __forceinline__ void to_rate2() {
#pragma unroll
    for (int j = 0; j < S / 2; ++j) v[j] = make_float2(rate2_of(v[j].x), rate2_of(v[j].y));
  }
};

// What a token does to one lane's states of one channel, h <- keep h + take, and what it reads out of them.
template <int S>
struct LaneToken {
  LaneStates<S> keep, take;
  __device__ __forceinline__ void make(const LaneStates<S>& rate2, float step, float in, const LaneStates<S>& b) {
#pragma unroll
    for (int j = 0; j < S / 2; ++j) {
      keep.v[j] = make_float2(exp2_fast(step * rate2.v[j].x), exp2_fast(step * rate2.v[j].y));
      take.v[j] = make_float2(in * b.v[j].x, in * b.v[j].y);
    }
  }
  // The lane's part of the sum over n.  `real`: how many of the lane's states there are; the others stay 0 (an infinite x times their
  // zero B would be NaN).
  template <bool PAD>
  __device__ __forceinline__ float go(LaneStates<S>& h, const LaneStates<S>& c, int real) const {
    float2 sum;
#pragma unroll
    for (int j = 0; j < S / 2; ++j) {
      h.v[j] = fma_f32x2(keep.v[j], h.v[j], take.v[j]);
      if (PAD) {
        if (2 * j >= real) h.v[j].x = 0.0f;
        if (2 * j + 1 >= real) h.v[j].y = 0.0f;
      }
      sum = j == 0 ? mul_f32x2(c.v[j], h.v[j]) : fma_f32x2(c.v[j], h.v[j], sum);
    }
    return sum.x + sum.y;
  }
};

// Four neighbouring channels of a row as they lie in memory: float32, two bfloat16 in each of the first two words, or one by one (SPREAD),
// a bfloat16 in each word, so that nothing has to wait for a read where rows cannot be read by four.
struct FourRaw { uint4 v; };

__device__ __forceinline__ FourRaw load_spread(const void* p, int dtype, bool wide, int left) {
  FourRaw r;
  r.v = make_uint4(0u, 0u, 0u, 0u);
  if (dtype == IFX_DT_F32) {
    const uint32_t* q = static_cast<const uint32_t*>(p);
    if (wide && left >= 4) return FourRaw{*reinterpret_cast<const uint4*>(q)};
    if (left > 0) r.v.x = q[0];
    if (left > 1) r.v.y = q[1];
    if (left > 2) r.v.z = q[2];
    if (left > 3) r.v.w = q[3];
  } else {
    const unsigned short* q = static_cast<const unsigned short*>(p);
    if (left > 0) r.v.x = q[0];
    if (left > 1) r.v.y = q[1];
    if (left > 2) r.v.z = q[2];
    if (left > 3) r.v.w = q[3];
  }
  return r;
}

template <bool SPREAD>
__device__ __forceinline__ float4 four_f32(const FourRaw& r, int dtype) {
  if (dtype == IFX_DT_F32) return make_float4(__uint_as_float(r.v.x), __uint_as_float(r.v.y), __uint_as_float(r.v.z), __uint_as_float(r.v.w));
  if (SPREAD) return make_float4(__uint_as_float(r.v.x << 16), __uint_as_float(r.v.y << 16), __uint_as_float(r.v.z << 16), __uint_as_float(r.v.w << 16));
  return make_float4(__uint_as_float(r.v.x << 16), __uint_as_float(r.v.x & 0xffff0000u), __uint_as_float(r.v.y << 16),
                     __uint_as_float(r.v.y & 0xffff0000u));
}

__device__ __forceinline__ void store_four(void* p, long long at, int dtype, bool wide, int left, const float (&y)[4]) {
  if (dtype == IFX_DT_F32) {
    float* q = static_cast<float*>(p) + at;
    if (wide && left >= 4) {
      *reinterpret_cast<float4*>(q) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) q[i] = y[i];
    }
  } else {
    __nv_bfloat16* q = static_cast<__nv_bfloat16*>(p) + at;
    if (wide && left >= 4) {
      __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
      *reinterpret_cast<uint2*>(q) = make_uint2(reinterpret_cast<uint32_t&>(lo), reinterpret_cast<uint32_t&>(hi));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) q[i] = __float2bfloat16_rn(y[i]);
    }
  }
}

// BYTES into shared memory, zeros where there is nothing to copy.  16 bytes pass L1 by: with all but 28 KB of an SM's memory shared, as every kernel
// here asks for, lines that wait for their data fill it (2,048 tokens of 7,168 channels 141 -> 123 us).
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool there) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(there ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(at), "l"(from), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}

template <int BYTES>
__device__ __forceinline__ FourRaw read_four(const void* from) {
  if constexpr (BYTES == 16) return FourRaw{*static_cast<const uint4*>(from)};
  const uint2 two = *static_cast<const uint2*>(from);
  return FourRaw{make_uint4(two.x, two.y, 0u, 0u)};
}

constexpr int kWalkers = 256, kWorkers = 256, kSpanThreads = kWalkers + kWorkers, kStepThreads = 128;
constexpr int kLaneStates = 4;             // of a channel in a lane

template <int LANES>
struct SpanTile {
  static constexpr int kChannels = kWalkers / LANES;                     // of a block
  static constexpr int kTokens = LANES == 1 ? 8 : LANES == 2 || LANES == 32 ? 16 : 32;
  static constexpr int kStates = kLaneStates * LANES;                    // with those that fill up
  static constexpr int kFours = (kTokens * kChannels + 4 * kWorkers - 1) / (4 * kWorkers);       // of a worker and tile
  static constexpr int kTogether = 4;                                    // tokens of a group
  // the lanes' sums [lane][token][channel]: a plane a lane, so placed that a warp's stores fall on different banks (up to 8 lanes)
  static constexpr int kPlane = kTokens * kChannels + (LANES < 8 ? 32 / LANES : 4);
  // floats of shared memory: steps and sums twice, B and C and what the workers fetch once a stage
  static constexpr int kStages = 3;                                      // tiles that are under way at once
  static constexpr int kSteps = 2 * kChannels * kTokens;
  static constexpr int kBC = 2 * kStates * kTokens;
  static constexpr int kRows = kWorkers * kFours;                        // fours of an operand and stage
};

// Bytes of shared memory, with four channels of x, z and of dt in `xb` and `db` bytes.
template <int LANES>
constexpr int span_bytes(int xb, int db) {
  using T = SpanTile<LANES>;
  return 4 * (2 * T::kSteps + T::kStages * T::kBC + 2 * LANES * T::kPlane) + T::kStages * T::kRows * (2 * xb + db);
}

// Four channels' sums over their lanes: neighbours first, then pairs of neighbours, and so on.
template <int LANES>
__device__ __forceinline__ void lanes_sum(const float* p, int plane, float (&out)[4]) {
  if constexpr (LANES == 1) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    out[0] = f.x; out[1] = f.y; out[2] = f.z; out[3] = f.w;
  } else {
    float more[4];
    lanes_sum<LANES / 2>(p, plane, out);
    lanes_sum<LANES / 2>(p + LANES / 2 * plane, plane, more);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] += more[j];
  }
}

// The request of a block: by the lengths of their spans, longest first, so that the last blocks to begin are short ones (more than 32: as
// they come).
__device__ __forceinline__ int request_by_length(const int* __restrict__ cu_seqlens, int requests, int place) {
  if (requests < 2 || requests > 32) return place;
  const int lane = threadIdx.x & 31;
  const int mine = lane < requests ? cu_seqlens[lane + 1] - cu_seqlens[lane] : -1;
  int before = 0;
  for (int r = 0; r < requests; ++r) {
    const int other = __shfl_sync(0xffffffffu, mine, r);
    before += other > mine || (other == mine && r < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < requests && before == place)) - 1;
}

// Spans of tokens.  A block has up to 256 / LANES channels of one request and goes through its tokens in tiles.  Eight warps walk: a thread has
// four states of a channel.  Eight other warps fetch (two tiles ahead), make steps and steps times x of the next tile, and of the tile before add
// up the lanes' sums over n, finish and store.
//
// Bound: the walk.  A token costs a channel as many exponentials as it has states (16 of them a clock and SM: 52 us for 2,048 tokens of 7,168 channels of
// 16 states, 65 with those of steps and gates); bytes would take 23.  Measured 123 us: a walking warp issues 24 instructions a token, four of which
// hold its exponential unit for eight clocks each, and a scheduler has two such warps, or one, beside two that fetch.  Of what was measured on the way
// (same sizes, us): walk and rows by the same warps 281; two states a lane 165 (shared memory gives a warp 128 bytes a clock, and what a token's B
// and C cost it is the same for two states as for four); when walkers apart took 131: two channels a thread 150, decays four tokens ahead instead of
// two 131, a quarter of the exponentials by a polynomial 146, twice the workers 131, half of them 142.
//
// By stretches (what `stretch` and `pass` say): where channels are few, a span's tokens are cut into stretches of `stretch`, a block each.
// The first pass walks the first stretch as it is, and of the others but the last only what they make of a state of zeros and how much of what was
// there they leave, which is one exponential of the steps' sum; both go to `ends`, [request][stretch][channels (states + 1)].  The second
// pass puts every stretch's first state together from those in front of it and walks again.
//
// XT, DT: the dtypes of x (and z and out) and of dt where all rows can be read by four channels; -1: as the arguments say.
template <int LANES, bool PAD, int XT, int DT>
__global__ void __launch_bounds__(kSpanThreads, 1) selective_span_kernel(const SelectiveArgs a) {
  using Tile = SpanTile<LANES>;
  constexpr int S = kLaneStates, CH = Tile::kChannels, TT = Tile::kTokens, NP = Tile::kStates, K = Tile::kFours, G = Tile::kTogether,
                PLANE = Tile::kPlane, ST = Tile::kStages;
  constexpr bool KNOWN = XT >= 0;
  extern __shared__ __align__(16) float span_s[];
  float2* const step_s = reinterpret_cast<float2*>(span_s);              // [2][TT][CH]: steps, and steps times x
  float* const bc_s = span_s + 2 * Tile::kSteps;                         // [ST][TT][2 NP]
  float* const y_s = bc_s + ST * Tile::kBC;                              // [2][LANES][PLANE]
  const int r = request_by_length(a.cu_seqlens, gridDim.y, blockIdx.y), k_stretch = blockIdx.z + (a.pass == 2);
  const int c0 = blockIdx.x * a.per_block, channels = min(a.channels, c0 + a.per_block);
  const int span = a.cu_seqlens[r + 1] - a.cu_seqlens[r];
  const long long begin = a.pass ? (long long)k_stretch * a.stretch : 0;
  const long long first = a.cu_seqlens[r] + begin;
  const bool last = !a.pass || span - begin <= a.stretch;                // nothing of the span lies behind
  const int n = (int)min((long long)span - begin, a.pass ? (long long)a.stretch : (long long)span);
  const bool local = a.pass == 1 && k_stretch > 0;                       // what it makes of zeros, without any output
  const int tiles = local && last ? 0 : (n + TT - 1) / TT;               // (n <= 0: none)
  float* const ends = a.ends + (long long)r * (gridDim.z + 1) * a.channels * (a.states + 1);   // (a grid has a stretch less than there are)
  if (threadIdx.x < kWalkers) {                                          // ---- the walk
    // neighbouring lanes have neighbouring channels and the same states: what they read of B and C is one address
    const int tid = threadIdx.x, part = tid % 32 / (32 / LANES), mine = tid / 32 * (32 / LANES) + tid % (32 / LANES), c = c0 + mine,
              real = c < channels ? a.states - part * S : 0;
    const bool idle = c0 + tid / 32 * (32 / LANES) >= channels;          // a warp without channels
    LaneStates<S> rate2, h;
    const long long at_c = (long long)c * a.states + part * S, end_size = (long long)a.channels * (a.states + 1);
    rate2.load(a.log_rate + at_c, real);
    rate2.to_rate2();
    pdl_wait();
    if (tiles <= 0) return;
    float* st = a.state + (long long)a.req_slot[r] * a.slot_stride + at_c;
    if (a.pass == 2) {                                                   // what the stretches in front leave
      h.load(ends + at_c, real);
      for (int k = 1; k < k_stretch; ++k) {
        const float* end = ends + k * end_size;
        const float steps = c < channels ? end[(long long)a.channels * a.states + c] : 0.0f;
        LaneStates<S> more;
        more.load(end + at_c, real);
#pragma unroll
        for (int j = 0; j < S / 2; ++j)
          h.v[j] = fma_f32x2(make_float2(exp2_fast(steps * rate2.v[j].x), exp2_fast(steps * rate2.v[j].y)), h.v[j], more.v[j]);
      }
    } else {
      h.load(st, local ? 0 : real);
    }
    float steps_sum = 0.0f;
    if (PAD) __syncthreads();
    __syncthreads();                                                     // tile 0 is there
    for (int i = 0; i < tiles; ++i) {
      if (idle) {
        __syncthreads();
        continue;
      }
      const int at = i & 1, groups = (min(TT, n - i * TT) + G - 1) / G;
      const float2* steps = step_s + at * TT * CH + mine;
      const float* bc = bc_s + i % ST * (TT * 2 * NP) + part * S;
      float* sums = y_s + (at * LANES + part) * PLANE + mine;
      if (local) {
        for (int g = 0; g < groups; ++g) {
          float2 step[G];
          LaneStates<S> b[G];
          LaneToken<S> token[G];
#pragma unroll
          for (int j = 0; j < G; ++j) {
            step[j] = steps[j * CH];
            b[j].load_wide(bc + j * 2 * NP);
          }
#pragma unroll
          for (int j = 0; j < G; ++j) token[j].make(rate2, step[j].x, step[j].y, b[j]);
#pragma unroll
          for (int j = 0; j < G; ++j) token[j].template go<PAD>(h, b[j], real);
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < G; ++j) sum += step[j].x;
          steps_sum += sum;
          steps += G * CH;
          bc += G * 2 * NP;
        }
        __syncthreads();
        continue;
      }
      // Pairs of tokens: of the one that goes through the states everything is there; of the next one, whose exponentials are made meanwhile, the
      // arguments; of the one behind it, what it is made of.
      struct Pair { LaneStates<S> keep[2], take[2], c[2]; } one, two;
      float2 step[2];
      LaneStates<S> b[2];
      auto read = [&](int q) {                                           // pair q from where the pointers are
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          step[j] = steps[(2 * q + j) * CH];
          b[j].load_wide(bc + (2 * q + j) * 2 * NP);
        }
      };
      auto refill = [&](Pair& p, int q) {                                // from what has been read: arguments in the place of decays
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int k = 0; k < S / 2; ++k) {
            p.keep[j].v[k] = make_float2(step[j].x * rate2.v[k].x, step[j].x * rate2.v[k].y);
            p.take[j].v[k] = make_float2(step[j].y * b[j].v[k].x, step[j].y * b[j].v[k].y);
          }
          p.c[j].load_wide(bc + (2 * q + j) * 2 * NP + NP);
        }
      };
      auto exponentials = [&](Pair& p, int j) {
#pragma unroll
        for (int k = 0; k < S / 2; ++k) p.keep[j].v[k] = make_float2(exp2_fast(p.keep[j].v[k].x), exp2_fast(p.keep[j].v[k].y));
      };
      using Yes = std::true_type;
      using No = std::false_type;
      // the pair q goes; `exps`: there is one behind it, `refills`: and one behind that, which takes its place
      auto go = [&](Pair& p, Pair& behind, int q, auto exps, auto refills) {
        float y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          LaneToken<S> t{p.keep[j], p.take[j]};
          if constexpr (decltype(exps)::value) exponentials(behind, j);
          y[j] = t.template go<PAD>(h, p.c[j], real);
        }
        if constexpr (decltype(refills)::value) {
          refill(p, q + 2);
          read(q + 3);                                                   // (behind a tile's last token: not used)
        }
        sums[2 * q * CH] = y[0];
        sums[(2 * q + 1) * CH] = y[1];
      };
      int pairs = (min(TT, n - i * TT) + 1) / 2;
      read(0);
      refill(one, 0);
      exponentials(one, 0);
      exponentials(one, 1);
      read(1);
      refill(two, 1);
      read(2);
#pragma unroll 1
      for (; pairs >= 4; pairs -= 2) {
        go(one, two, 0, Yes{}, Yes{});
        go(two, one, 1, Yes{}, Yes{});
        steps += 4 * CH;
        bc += 4 * 2 * NP;
        sums += 4 * CH;
      }
      if (pairs == 3) {
        go(one, two, 0, Yes{}, Yes{});
        go(two, one, 1, Yes{}, No{});
        go(one, two, 2, No{}, No{});
      } else if (pairs == 2) {
        go(one, two, 0, Yes{}, No{});
        go(two, one, 1, No{}, No{});
      } else {
        go(one, two, 0, No{}, No{});
      }
      __syncthreads();
    }
    if (last) {
      h.store(st, real);
    } else if (a.pass == 1) {
      float* end = ends + k_stretch * end_size;
      h.store(end + at_c, real);
      if (part == 0 && c < channels) end[(long long)a.channels * a.states + c] = steps_sum;
    }
    return;
  }
  // ---- the others: four channels of some of a tile's tokens each
  const int x_dtype = KNOWN ? XT : a.x_dtype, dt_dtype = KNOWN ? DT : a.dt_dtype, out_dtype = KNOWN ? XT : a.out_dtype;
  const bool wide_out = KNOWN || (a.wide & 16);
  const int tid = threadIdx.x - kWalkers, f4 = 4 * (tid % (CH / 4)), ft = tid / (CH / 4);
  // channels of the four that there are (with known rows all or none), and none for threads behind a tile's tokens
  const int left = ft < TT ? channels - c0 - f4 : 0;
  constexpr int kStride = kWorkers / (CH / 4);                           // tokens from one of a thread's to the next
  static_assert(K == 1 || K * kStride == TT, "a tile's tokens are shared out evenly");
  float4 bias = make_float4(0.0f, 0.0f, 0.0f, 0.0f), skip = bias;
  if (a.bias) bias = four_f32<true>(load_spread(a.bias + c0 + f4, IFX_DT_F32, false, left), IFX_DT_F32);
  if (a.skip) skip = four_f32<true>(load_spread(a.skip + c0 + f4, IFX_DT_F32, false, left), IFX_DT_F32);
  pdl_wait();
  if (tiles <= 0) return;
  if constexpr (PAD) {
    for (int i = tid; i < ST * TT * 2 * NP; i += kWorkers) bc_s[i] = 0.0f;
    __syncthreads();
  }
  // A thread copies what it will need of a tile into places of its own; only B and C are for all.
  constexpr int XB = XT == IFX_DT_BF16 ? 8 : 16, DB = DT == IFX_DT_BF16 ? 8 : 16, kStage = K * kWorkers * (2 * XB + DB);
  char* const stages = reinterpret_cast<char*>(y_s + 2 * LANES * PLANE);        // [ST]: x [K][worker], z, dt
  auto place = [&](char* stage, int operand, int k) {
    return stage + (operand == 2 ? (2 * K + k) * kWorkers * XB - k * kWorkers * (XB - DB) + tid * DB : ((operand * K + k) * kWorkers + tid) * XB);
  };
  const int x_size = x_dtype == IFX_DT_F32 ? 4 : 2, dt_size = dt_dtype == IFX_DT_F32 ? 4 : 2, out_size = out_dtype == IFX_DT_F32 ? 4 : 2;
  // the thread's first token of the tile to fetch, or to store, and from one of its tokens to the next
  const char* from_x = static_cast<const char*>(a.x) + ((first + ft) * a.ld_x + c0 + f4) * x_size;
  const char* from_z = static_cast<const char*>(a.z) + ((first + ft) * a.ld_z + c0 + f4) * x_size;
  const char* from_dt = static_cast<const char*>(a.dt) + ((first + ft) * a.ld_dt + c0 + f4) * dt_size;
  char* to_out = static_cast<char*>(a.out) + ((first + ft) * a.channels + c0 + f4) * out_size;
  const long long row_x = a.ld_x * x_size, row_z = a.ld_z * x_size, row_dt = a.ld_dt * dt_size, row_out = (long long)a.channels * out_size;
  const bool gated = a.z != nullptr && !local;
  // B and C by 16 bytes: a worker's pieces of a tile, which lie as in shared memory but for the distance between rows
  constexpr int kPieces = (TT * NP / 2 + kWorkers - 1) / kWorkers, kPieceRows = kWorkers / (NP / 2) > 0 ? kWorkers / (NP / 2) : 1;
  static_assert(PAD || kPieces * kWorkers == TT * NP / 2 || kPieces == 1, "pieces are shared out evenly");
  const int piece_row = tid / (NP / 2), piece_col = tid % (NP / 2) * 4;
  const float* from_bc = a.bc + (first + piece_row) * a.ld_bc + piece_col;
  FourRaw hold[KNOWN ? 1 : K][3];                                        // rows that cannot be copied by four: a tile's, on their way
  int held = -1;                                                         // its stage
  auto fetch = [&](int t0, int to) {                                     // one group of copies
    const bool whole = t0 + TT <= n;
    if (!PAD && (a.wide & 8)) {
      if (kPieces > 1 || tid < TT * NP / 2) {
        float* const to_bc = bc_s + to * Tile::kBC + 4 * tid;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const bool there = whole || t0 + piece_row + k * kPieceRows < n;
          copy_async<16>(to_bc + 4 * k * kWorkers, there ? from_bc + k * kPieceRows * a.ld_bc : a.bc, there);
        }
      }
      from_bc += TT * a.ld_bc;
    } else {
      for (int i = tid; i < TT * 2 * a.states; i += kWorkers) {
        const int t = i / (2 * a.states), j = i % (2 * a.states);
        copy_async<4>(bc_s + to * Tile::kBC + t * 2 * NP + (j < a.states ? j : NP + j - a.states),
                      a.bc + (first + min(t0 + t, n - 1)) * a.ld_bc + j, t0 + t < n);
      }
    }
    if (left > 0) {
      char* const stage = stages + to * kStage;
      if constexpr (!KNOWN) {                                            // what was asked for a tile ago goes to its place
        if (held >= 0)
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < 3; ++j) *reinterpret_cast<uint4*>(place(stages + held * kStage, j, k)) = hold[k][j].v;
        held = to;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!whole && t0 + ft + k * kStride >= n) break;
        if constexpr (KNOWN) {
          copy_async<DB>(place(stage, 2, k), from_dt + k * kStride * row_dt, true);
          copy_async<XB>(place(stage, 0, k), from_x + k * kStride * row_x, true);
          if (gated) copy_async<XB>(place(stage, 1, k), from_z + k * kStride * row_z, true);
        } else {
          hold[k][2] = load_spread(from_dt + k * kStride * row_dt, dt_dtype, a.wide & 2, left);
          hold[k][0] = load_spread(from_x + k * kStride * row_x, x_dtype, a.wide & 1, left);
          if (gated) hold[k][1] = load_spread(from_z + k * kStride * row_z, x_dtype, a.wide & 4, left);
        }
      }
      from_x += TT * row_x;
      from_z += TT * row_z;
      from_dt += TT * row_dt;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto make = [&](int t0, int buffer, int at) {
    if (left <= 0) return;
    char* const stage = stages + at * kStage;
    float4* const to = reinterpret_cast<float4*>(step_s + (buffer * TT + ft) * CH + f4);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float4 x = four_f32<!KNOWN>(read_four<XB>(place(stage, 0, k)), x_dtype), raw = four_f32<!KNOWN>(read_four<DB>(place(stage, 2, k)), dt_dtype);
      const float4 step = make_float4(softplus_f32(raw.x + bias.x), softplus_f32(raw.y + bias.y), softplus_f32(raw.z + bias.z), softplus_f32(raw.w + bias.w));
      to[k * kStride * CH / 2] = make_float4(step.x, step.x * x.x, step.y, step.y * x.y);
      to[k * kStride * CH / 2 + 1] = make_float4(step.z, step.z * x.z, step.w, step.w * x.w);
    }
    if (t0 + TT > n)                                                     // a token that is not there changes nothing
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (t0 + ft + k * kStride >= n) to[k * kStride * CH / 2] = to[k * kStride * CH / 2 + 1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  };
  auto finish = [&](int t0, int buffer, int at) {
    if (left <= 0) return;
    char* const stage = stages + at * kStage;
    const float* const sums = y_s + buffer * LANES * PLANE + ft * CH + f4;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (t0 + TT > n && t0 + ft + k * kStride >= n) break;
      const float4 x = four_f32<!KNOWN>(read_four<XB>(place(stage, 0, k)), x_dtype);
      float out[4];
      lanes_sum<LANES>(sums + k * kStride * CH, PLANE, out);
      if (a.skip) {                                                      // (no skip is not one of zero: x may be infinite)
        out[0] = fmaf(skip.x, x.x, out[0]);
        out[1] = fmaf(skip.y, x.y, out[1]);
        out[2] = fmaf(skip.z, x.z, out[2]);
        out[3] = fmaf(skip.w, x.w, out[3]);
      }
      if (gated) {
        const float4 z = four_f32<!KNOWN>(read_four<XB>(place(stage, 1, k)), x_dtype);
        out[0] *= silu_f32(z.x);
        out[1] *= silu_f32(z.y);
        out[2] *= silu_f32(z.z);
        out[3] *= silu_f32(z.w);
      }
      store_four(to_out + k * kStride * row_out, 0, out_dtype, wide_out, KNOWN ? 4 : left, out);
    }
    to_out += TT * row_out;
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) fetch(s * TT, s);
  asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
  make(0, 0, 0);
  __syncthreads();
  for (int i = 0, stage = 0; i < tiles; ++i) {
    const int t0 = i * TT, next = stage + 1 == ST ? 0 : stage + 1;
    fetch(t0 + (ST - 1) * TT, stage == 0 ? ST - 1 : stage - 1);          // where tile i - 1 was, which everybody is through with
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");    // tile i + 1 is there
    if (i + 1 < tiles) make(t0 + TT, (i + 1) & 1, next);
    __syncthreads();                                                     // tile i has been walked, tile i + 1 can be
    if (!local) finish(t0, i & 1, stage);
    stage = next;
  }
}

// One token a request at most: a thread has four states of a channel of Q requests, whose rates it makes once; all its reads are under way
// before the first is looked at (dtypes that a branch chooses are turned into float32 behind the last of them).  What there is once a
// channel (the step, the gate, the skip, the result's way out) is done by one lane for each request, not by all of them (us: 15.0 for
// 15.7; 24 requests 5.3 for 5.9, before steps and gates carried what their exponential's argument was rounded by).  WIDE: states, rates, B and C four at a time.  Bound by the states' way in and out: 64 requests of
// 7,168 channels of 16 states, 64 MB, 15.2 us, 4.2 TB/s.
template <int LANES, bool PAD, bool WIDE, int Q>
__global__ void __launch_bounds__(kStepThreads) selective_step_kernel(const SelectiveArgs a, int requests) {
  constexpr int S = kLaneStates, CH = kStepThreads / LANES;
  const int r0 = blockIdx.y * Q, part = threadIdx.x % LANES, c_mine = blockIdx.x * CH + threadIdx.x / LANES, real = a.states - part * S;
  const int c = min(c_mine, a.channels - 1);                 // (threads behind the last channel read it, and store nothing)
  pdl_launch_dependents();
  LaneStates<S> rate2, h[Q], b[Q], c_[Q];
  auto get = [&](LaneStates<S>& to, const float* from) {
    if (WIDE) to.load_wide(from);
    else to.load(from, real);
  };
  get(rate2, a.log_rate + (long long)c * a.states + part * S);
  const float bias = a.bias ? a.bias[c] : 0.0f, skip = a.skip ? a.skip[c] : 0.0f;
  // what there is once a channel is done for request `own` alone, and handed to the channel's other lanes
  const int own = part % Q;
  int t[Q], t_own = 0;
  bool any[Q], any_own = false;
  float* st[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int r = min(r0 + q, requests - 1);
    t[q] = a.cu_seqlens[r];
    any[q] = r0 + q < requests && a.cu_seqlens[r + 1] > t[q];
    st[q] = a.state + (long long)a.req_slot[r] * a.slot_stride + (long long)c * a.states + part * S;
    if (q == own) { t_own = t[q]; any_own = any[q]; }
  }
  pdl_wait();
  uint32_t x_raw = 0u, dt_raw = 0u, z_raw = 0u;
  if (any_own) {
    x_raw = load_raw(a.x, t_own * a.ld_x + c, a.x_dtype);
    dt_raw = load_raw(a.dt, t_own * a.ld_dt + c, a.dt_dtype);
    if (a.z) z_raw = load_raw(a.z, t_own * a.ld_z + c, a.x_dtype);
  }
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if (!any[q]) continue;                                               // (the same for a whole block)
    get(h[q], st[q]);
    get(b[q], a.bc + t[q] * a.ld_bc + part * S);
    get(c_[q], a.bc + t[q] * a.ld_bc + a.states + part * S);
  }
  rate2.to_rate2();
  const float x = raw_f32(x_raw, a.x_dtype), step = softplus_f32(raw_f32(dt_raw, a.dt_dtype) + bias), in = step * x;
  float y_own = 0.0f;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if (!any[q]) continue;
    const float step_q = Q == 1 ? step : __shfl_sync(0xffffffffu, step, q, LANES), in_q = Q == 1 ? in : __shfl_sync(0xffffffffu, in, q, LANES);
    LaneToken<S> token;
    token.make(rate2, step_q, in_q, b[q]);
    float y = token.template go<PAD>(h[q], c_[q], real);
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (q == own) y_own = y;
    if (c_mine < a.channels) {
      if (WIDE) h[q].store_wide(st[q]);
      else h[q].store(st[q], real);
    }
  }
  if (part >= Q || !any_own || c_mine >= a.channels) return;
  if (a.skip) y_own = fmaf(skip, x, y_own);
  if (a.z) y_own *= silu_f32(raw_f32(z_raw, a.x_dtype));
  const long long at = (long long)t_own * a.channels + c;
  if (a.out_dtype == IFX_DT_F32) static_cast<float*>(a.out)[at] = y_own;
  else static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(y_own);
}

struct SelectiveInputsArgs {
  const void* rows; long long ld; int dtype, splits; size_t split_stride;
  const float* w_low; const float* w_b; const float* w_c;      // null: that part is not normed
  float eps;
  void* low; int low_dtype;
  float* bc;
  int T, rank, states;
};

// A warp a row: a lane reads columns lane, lane + 32, ... (PER of them at most) before it looks at the first, and all three parts' sums of
// squares go through one chain of exchanges.  Bound by latency (few rows), then by the rows' way in and out.
template <int PER>
__global__ void __launch_bounds__(128) selective_inputs_kernel(const SelectiveInputsArgs a) {
  const int lane = threadIdx.x & 31, width = a.rank + 2 * a.states, behind_b = a.rank + a.states;
  const long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  const bool normed = a.w_low || a.w_b || a.w_c;
  float w[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = lane + 32 * k;
    w[k] = 1.0f;
    if (normed && i < width) {
      if (i < a.rank) { if (a.w_low) w[k] = a.w_low[i]; }
      else if (i < behind_b) { if (a.w_b) w[k] = a.w_b[i - a.rank]; }
      else if (a.w_c) w[k] = a.w_c[i - behind_b];
    }
  }
  pdl_wait();
  if (t >= a.T) return;
  float v[PER];
  uint32_t raw[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) raw[k] = lane + 32 * k < width ? load_raw(a.rows, t * a.ld + lane + 32 * k, a.dtype) : 0u;
#pragma unroll
  for (int k = 0; k < PER; ++k) v[k] = raw_f32(raw[k], a.dtype);
  for (int s = 1; s < a.splits; ++s) {                                   // (in the order of the slices)
    const float* more = static_cast<const float*>(a.rows) + s * a.split_stride + t * a.ld + lane;
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (lane + 32 * k < width) v[k] += more[32 * k];
  }
  float scale[3] = {1.0f, 1.0f, 1.0f};
  if (normed) {
    float sum[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = lane + 32 * k;
      const float q = v[k] * v[k];
      if (i < a.rank) sum[0] += q;
      else if (i < behind_b) sum[1] += q;
      else sum[2] += q;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int j = 0; j < 3; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
    if (a.w_low) scale[0] = rsqrtf(sum[0] / (float)a.rank + a.eps);
    if (a.w_b) scale[1] = rsqrtf(sum[1] / (float)a.states + a.eps);
    if (a.w_c) scale[2] = rsqrtf(sum[2] / (float)a.states + a.eps);
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = lane + 32 * k;
    if (i >= width) continue;
    const float y = normed ? v[k] * scale[i < a.rank ? 0 : i < behind_b ? 1 : 2] * w[k] : v[k];
    if (i >= a.rank) a.bc[t * 2 * a.states + i - a.rank] = y;
    else if (a.low_dtype == IFX_DT_F32) static_cast<float*>(a.low)[t * a.rank + i] = y;
    else static_cast<__nv_bfloat16*>(a.low)[t * a.rank + i] = __float2bfloat16_rn(y);
  }
}

// Wide rows: a warp keeps one in shared memory between the sum of squares and the result.
__global__ void __launch_bounds__(128) selective_inputs_wide_kernel(const SelectiveInputsArgs a) {
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

static int lanes_of(int states) {
  int lanes = 1;
  while (lanes * kLaneStates < states) lanes <<= 1;
  return lanes;
}

// Into how many stretches the longest span is cut at most (0: spans are walked whole).  Two passes of stretches side by side take 2 / stretches of
// the walk, and a launch; all blocks of a pass run at once.  us, whole and by stretches, one span: 1,024 channels of 16 states, 4,000 tokens
// 176 / 59; 300 16.3 / 15.3; 2,048 channels, 2,048 tokens 94 / 59, 500 25.6 / 21.6; 512 channels, 200 tokens 13.2 / 15.1; 4,096 channels (three stretches), 2,048
// tokens 100 / 97, 512 27.1 / 30.2.
static int stretches_of(int channels, int states, int requests, int max_span) {
  const long long per_block = kWalkers / lanes_of(states), blocks = (channels + per_block - 1) / per_block * requests;
  const long long most = 148 / blocks + 1;
  return most >= 4 && max_span >= 256 ? (int)most : 0;
}

template <int LANES, bool PAD>
static int launch_selective(SelectiveArgs a, int requests, int max_span, int stretches, cudaStream_t stream) {
  if (max_span == 1) {
    constexpr int kChannels = kStepThreads / LANES;
    const long long blocks = (a.channels + kChannels - 1) / kChannels;
    const bool wide = !PAD && (a.wide & 104) == 104;
    // two requests a thread share its rates; with few requests one, for the shorter way (us, one and two a thread, 16 states, read from beyond L2: 1,024
    // channels 12 requests 2.6 / 2.3, 24 2.9 / 3.2, 64 4.9 / 3.8; 2,048 8 2.8 / 2.9, 12 2.9 / 3.1, 64 7.6 / 5.9; 4,096 8 3.2 / 3.2, 16 4.7 / 3.7;
    // 7,168 4 3.1 / 3.0, 8 4.3 / 3.6, 12 5.4 / 4.5, 64 20.5 / 15.8)
    constexpr int kMost = LANES >= 2 ? 2 : 1;
    const int each = requests >= 12 ? kMost : 1;
    auto kernel = each == kMost ? (wide ? selective_step_kernel<LANES, PAD, !PAD, kMost> : selective_step_kernel<LANES, PAD, false, kMost>)
                                : (wide ? selective_step_kernel<LANES, PAD, !PAD, 1> : selective_step_kernel<LANES, PAD, false, 1>);
    return launch_pdl(kernel, dim3((unsigned)blocks, (unsigned)((requests + each - 1) / each)), dim3(kStepThreads), 0, stream, 1, a, requests);
  }
  using Tile = SpanTile<LANES>;
  constexpr int F = IFX_DT_F32, B = IFX_DT_BF16;
  auto kernel = selective_span_kernel<LANES, PAD, -1, -1>;
  int bytes = span_bytes<LANES>(16, 16);
  if ((a.wide & 19) == 19 && (!a.z || (a.wide & 4)) && a.channels % 4 == 0 && a.out_dtype == a.x_dtype) {
    kernel = a.x_dtype == F ? (a.dt_dtype == F ? selective_span_kernel<LANES, PAD, F, F> : selective_span_kernel<LANES, PAD, F, B>)
                            : (a.dt_dtype == F ? selective_span_kernel<LANES, PAD, B, F> : selective_span_kernel<LANES, PAD, B, B>);
    bytes = span_bytes<LANES>(a.x_dtype == F ? 16 : 8, a.dt_dtype == F ? 16 : 8);
  }
  static_assert(span_bytes<LANES>(16, 16) <= 227 * 1024, "shared memory of a block");
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return (int)e;
  const unsigned full = (unsigned)((a.channels + Tile::kChannels - 1) / Tile::kChannels);
  if (stretches) {
    a.stretch = ((max_span + stretches - 1) / stretches + Tile::kTokens - 1) / Tile::kTokens * Tile::kTokens;
    const unsigned count = (unsigned)((max_span + a.stretch - 1) / a.stretch);
    for (a.pass = 1; a.pass <= 2; ++a.pass) {
      const int rc = launch_pdl(kernel, dim3(full, (unsigned)requests, count - 1), dim3(kSpanThreads), bytes, stream, 1, a);
      if (rc) return rc;
    }
    return 0;
  }
  // One request: no more blocks than the rounds of 148 that full ones take, but with as few channels as that allows (4,096 channels of 16
  // states, 2,048 tokens: 131 -> 100 us).  With several, whose lengths differ, smaller blocks only take longer in all (700 tokens of three, 2,048 of 32
  // states: 22.8 -> 39.5).
  constexpr int kLeast = 32 / LANES > 4 ? 32 / LANES : 4;                // a warp's channels, and a worker's
  if (requests == 1) {
    const long long rounds = (full + 147) / 148;
    while (a.per_block > kLeast && (a.channels + a.per_block - kLeast - 1) / (a.per_block - kLeast) <= rounds * 148) a.per_block -= kLeast;
  }
  const unsigned blocks = (unsigned)((a.channels + a.per_block - 1) / a.per_block);
  return launch_pdl(kernel, dim3(blocks, (unsigned)requests), dim3(kSpanThreads), bytes, stream, 1, a);
}

static bool known_dtype(int d) { return d == IFX_DT_F32 || d == IFX_DT_BF16; }

// Floats that spans walked by stretches need (0: they are walked whole), for a step of so many requests whose longest span has max_span tokens.
extern "C" long long ifx_selective_scan_scratch(int num_requests, int max_span, int channels, int states) {
  if (num_requests <= 0 || num_requests > 65535 || max_span <= 1 || channels <= 0 || states <= 0 || states > 128) return 0;
  return stretches_of(channels, states, num_requests, max_span) * (long long)num_requests * channels * (states + 1);
}

// Row strides in elements.  x and z share a dtype; bc: float32 rows of B | C; state: float32, slots slot_stride floats apart.
// num_tokens: rows of x; cu_seqlens does not go beyond them.  A request without tokens keeps its state.  scratch: with scratch_floats of
// ifx_selective_scan_scratch long spans may go by stretches, whose sums depend on where a span begins and on the step's other spans (their number says
// whether there are stretches, the longest how long these are); null and 0: they do not.
extern "C" int ifx_selective_scan(const void* x, long long ld_x, int x_dtype, const void* dt, long long ld_dt, int dt_dtype, const float* bc,
                                  long long ld_bc, const void* z, long long ld_z, const float* log_rate, const float* bias, const float* skip,
                                  float* state, long long slot_stride, const int* req_slot, const int* cu_seqlens, void* out, int out_dtype,
                                  int num_requests, int num_tokens, int max_span, int channels, int states, float* scratch,
                                  long long scratch_floats, cudaStream_t stream) {
  if (num_requests < 0 || num_tokens < 0 || max_span < 0 || channels <= 0 || states <= 0) return IFX_E_BADARG;
  if (!known_dtype(x_dtype) || !known_dtype(dt_dtype) || !known_dtype(out_dtype)) return IFX_E_DTYPE;
  if (states > 128 || num_requests > 65535) return IFX_E_TOOBIG;
  if (num_requests == 0 || num_tokens == 0 || max_span == 0) return 0;
  if (ld_x < channels || ld_dt < channels || (z && ld_z < channels) || ld_bc < 2 * states || slot_stride < (long long)channels * states)
    return IFX_E_BADARG;
  if (!x || !dt || !bc || !log_rate || !state || !req_slot || !cu_seqlens || !out) return IFX_E_BADARG;
  auto four = [](const void* p, long long ld, int dtype) {
    return (uintptr_t)p % (dtype == IFX_DT_F32 ? 16 : 8) == 0 && ld % 4 == 0;
  };
  const int wide = (four(x, ld_x, x_dtype) ? 1 : 0) | (four(dt, ld_dt, dt_dtype) ? 2 : 0) | (z && four(z, ld_z, x_dtype) ? 4 : 0) |
                   (four(bc, ld_bc, IFX_DT_F32) && states % 4 == 0 ? 8 : 0) | (four(out, channels, out_dtype) ? 16 : 0) |
                   (four(state, slot_stride, IFX_DT_F32) ? 32 : 0) | ((uintptr_t)log_rate % 16 == 0 ? 64 : 0);
  SelectiveArgs a{x, ld_x, x_dtype, dt, ld_dt, dt_dtype, bc, ld_bc, z, ld_z, log_rate, bias, skip, state, slot_stride, req_slot, cu_seqlens,
                        out, out_dtype, channels, states, 0, 0, 0, scratch, wide};
  const int lanes = lanes_of(states);
  a.per_block = kWalkers / lanes;
  const int stretches = scratch_floats > 0 ? stretches_of(channels, states, num_requests, max_span) : 0;
  if (stretches && (!scratch || scratch_floats < stretches * (long long)num_requests * channels * (states + 1))) return IFX_E_BADARG;
  const bool pad = states != lanes * kLaneStates;
#define IFX_SELECTIVE(L)                                                                        \
  return pad ? launch_selective<L, true>(a, num_requests, max_span, stretches, stream)          \
             : launch_selective<L, false>(a, num_requests, max_span, stretches, stream)
  switch (lanes) {
    case 1: IFX_SELECTIVE(1);
    case 2: IFX_SELECTIVE(2);
    case 4: IFX_SELECTIVE(4);
    case 8: IFX_SELECTIVE(8);
    case 16: IFX_SELECTIVE(16);
    default: IFX_SELECTIVE(32);
  }
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
  if (width <= 512) {
    auto kernel = width <= 64 ? selective_inputs_kernel<2> : width <= 128 ? selective_inputs_kernel<4> : width <= 256 ? selective_inputs_kernel<8>
                                                                                                                 : selective_inputs_kernel<16>;
    return launch_pdl(kernel, dim3((unsigned)((T + 3) / 4)), dim3(128), 0, stream, 1, a);
  }
  const int warps = width <= 3000 ? 4 : 1;                       // of at most 48 KB of rows a block
  return launch_pdl(selective_inputs_wide_kernel, dim3((unsigned)((T + warps - 1) / warps)), dim3(32 * warps), (size_t)warps * width * 4, stream, 1, a);
}
