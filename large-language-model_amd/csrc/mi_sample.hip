// mi_sample.hip -- one token for each row of logits, by temperature, top-k, top-p and min-p, gfx950.
//
// With the tokens of a row ordered by (logit descending, index ascending), each of the three
// filters keeps a run from the front, so what is kept is fixed by one border: a logit, and how many
// of the tokens equal to it.  No sort is needed to find it:
//   1. a histogram over the distance from the row's maximum, SMP_BINS bins evenly over the distances
//      that can weigh anything, counts tokens (top-k) or sums weights (top-p);
//   2. a scan over the bins finds the one in which the border lies;
//   3. that bin's tokens (1/1000 of the row) go to LDS, where each finds its rank among them; where a
//      top-k keeps few, they all go there, and the row is not read again.
// A bin that holds more than SMP_LIST of them (a row of few distinct logits) is halved by its logits'
// bits instead, over the row, until one value is left.
//
// Weights w = 2^y, y = (x - max) log2(e) / T, are computed in 64 bits and held as integers, w * 2^shift,
// so every sum is exact: it is the same whatever order atomics and waves add in, and a border is never
// moved by rounding.  A weight below half of 2^-shift counts as nothing: u = 0, one of 2^24 numbers,
// then does not draw a token whose chance is 1e-20.  64 bits cost no more than 32 here (a 64-lane
// instruction takes four cycles either way); 2^y is a table of 32 steps in LDS, a polynomial of degree 5
// on what is left, and an addition that leaves the rounded integer in the low bits.  Tokens that a
// border has left are gathered 64 at a time before they are weighed: of a nucleus of 5 % of the
// vocabulary nearly every 64 tokens hold one, and weighing costs more than the rest of a pass.
//
// One workgroup a row, each wave a run of it.  A pass reads the row again, from the caches: held in
// registers it would need every pass unrolled over them, more code than the instruction cache holds.
// Bound by the passes' instructions, 0.2 us for each one an element at 32000 logits on a CU.
#include <hip/hip_runtime.h>
#include <math.h>

#include <type_traits>

#include "mi_gemm_device.hpp"
#include "mi_host.hpp"

namespace mig {
namespace {

constexpr int SMP_BINS = 1024;
constexpr int SMP_LIST = 1024;        // tokens of a bin that are ranked in LDS
constexpr int SMP_FEW = 256;          // tokens that are handled in LDS altogether
constexpr int SMP_GATHER = 4;         // logits that a lane weighs at a time: its waits for each overlap

struct SampleParams {
  const void* logits;
  int64_t ld;
  int vocab, shift;
  int layers;  // 16-byte vectors of a lane
  const float* u;
  int32_t* tokens;
  float* probs;
  mi_sampling how;
};

// Keys order as finite floats do (halving a range of values by their bits).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

template <bool BF16>
__device__ __forceinline__ float smp_elem(const u32x4_t& v, int e) {
  if constexpr (BF16) return (e & 1) ? __uint_as_float(v[e >> 1] & 0xffff0000u) : bf16_bits_to_f32(v[e >> 1]);
  else return __uint_as_float(v[e]);
}

// Elements j .. of a row of V as one vector; past the row's end -inf.
template <bool BF16, bool ALIGNED>
__device__ __forceinline__ u32x4_t smp_load(const void* row, int j, int V) {
  constexpr int EV = BF16 ? 8 : 4;
  const uint32_t none = BF16 ? 0xff80ff80u : 0xff800000u;
  u32x4_t v = {none, none, none, none};
  if (ALIGNED && j + EV <= V) return *(const u32x4_t*)((const char*)row + (int64_t)j * (BF16 ? 2 : 4));
#pragma unroll
  for (int e = 0; e < EV; ++e) {
    if (j + e >= V) continue;
    if constexpr (BF16) {
      const uint32_t h = ((const uint16_t*)row)[j + e];
      v[e >> 1] = (e & 1) ? (v[e >> 1] & 0xffffu) | h << 16 : (v[e >> 1] & 0xffff0000u) | h;
    } else {
      v[e] = ((const uint32_t*)row)[j + e];
    }
  }
  return v;
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  return v;
}

template <int WAVES>
struct SampleShared {
  uint64_t bins[SMP_BINS];
  uint64_t weights[SMP_LIST];
  float list[SMP_LIST];
  int index[SMP_LIST];
  double pow32[32];  // 2^(j/32)
  float pending[WAVES][64 * (SMP_GATHER + 8)];
  uint64_t wave_sum[WAVES];
  uint32_t wave_cnt[WAVES];
  float wave_mx[WAVES], wave_mn[WAVES];
  uint64_t above, upto;
  uint32_t n_list, bin;
  float border;
  uint32_t ties;
};

template <int TH, bool BF16, bool ALIGNED>
__global__ void __launch_bounds__(TH) sample_kernel(SampleParams p) {
  constexpr int EV = BF16 ? 8 : 4, WAVES = TH / 64;
  __shared__ SampleShared<WAVES> sh;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int V = p.vocab, layers = p.layers;
  const void* x = (const char*)p.logits + (int64_t)row * p.ld * (BF16 ? 2 : 4);
  // this wave's run of the row: layer i holds elements first + (64 i + lane) EV ..; a whole number of
  // layers covers it, so runs of the last waves may lie past its end (the sum stays below 2^25)
  const int first = wave * layers * 64 * EV + lane * EV;
  auto layer = [&](int i) __attribute__((always_inline)) {
    return smp_load<BF16, ALIGNED>(x, first + 64 * EV * i, V);
  };
  // f(i, vector) over this lane's vectors, the next one on its way; f returns whether to go on (the
  // same in all lanes)
  auto each_vector = [&](auto f) __attribute__((always_inline)) {
    u32x4_t v = layer(0);
    for (int i = 0; i < layers; ++i) {
      const u32x4_t next = layer(i + 1);
      if (!f(i, v)) break;
      v = next;
    }
  };
  auto each = [&](auto f) __attribute__((always_inline)) {
    each_vector([&](int, const u32x4_t& v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < EV; ++e) f(smp_elem<BF16>(v, e));
      return true;
    });
  };

  float T = p.how.temperature ? p.how.temperature[row] : p.how.temperature_all;
  const int top_k = p.how.top_k ? p.how.top_k[row] : p.how.top_k_all;
  const float top_p = p.how.top_p ? p.how.top_p[row] : p.how.top_p_all;
  const float min_p = p.how.min_p ? p.how.min_p[row] : p.how.min_p_all;
  const float u = p.u[row];
  const bool greedy = !(T > 0.0f) || top_k == 1;
  if (tid < 32) sh.pow32[tid] = exp2(tid * 0.03125);

  // largest and smallest logit above -inf (NaN is neither)
  float mx = -INFINITY, mn = INFINITY;
  each([&](float v) __attribute__((always_inline)) {
    mx = fmaxf(mx, v);
    mn = fminf(mn, v > -INFINITY ? v : INFINITY);
  });
  const float lane_mx = mx;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    mn = fminf(mn, __shfl_xor(mn, o, 64));
  }
  if (lane == 0) sh.wave_mx[wave] = mx, sh.wave_mn[wave] = mn;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    mx = fmaxf(mx, sh.wave_mx[w]);
    mn = fminf(mn, sh.wave_mn[w]);
  }
  if (mx == -INFINITY) {
    if (tid == 0) {
      p.tokens[row] = -1;
      if (p.probs) p.probs[row] = 0.0f;
    }
    return;
  }
  if (greedy) {
    if (tid == 0) sh.bin = V;
    __syncthreads();
    each_vector([&](int i, const u32x4_t& v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = EV - 1; e >= 0; --e)
        if (smp_elem<BF16>(v, e) == mx) atomicMin(&sh.bin, (uint32_t)(first + 64 * EV * i + e));
      return true;
    });
    __syncthreads();
    if (tid == 0) {
      p.tokens[row] = (int)sh.bin;
      if (p.probs) p.probs[row] = 1.0f;
    }
    return;
  }

  // weights of logits up to a finite maximum
  const double c = 1.4426950408889634074 / (double)T;
  const double c32 = 32.0 * c, mxd = (double)mx;
  const double to_bits = 1.5 * (double)(uint64_t{1} << (52 - p.shift));  // w + this: w * 2^shift in the low bits
  auto weight_of = [&](float v) __attribute__((always_inline)) {  // as a 64-bit float
    const double y = max(((double)v - mxd) * c32, -2048.0);  // 32 y; 2^-64 rounds to nothing
    const double t = y + 6755399441055744.0;                 // 1.5 * 2^52: rounded, in the low bits
    const int n = (int)(uint32_t)__double_as_longlong(t);
    const double z = y - (t - 6755399441055744.0);           // |z| <= 1/2, of 1/32
    // 2^(z/32) = sum (z ln 2 / 32)^k / k!, past k = 5 below 2^-48
    double q = 3.9737099845494154e-11;
    q = fma(q, z, 9.172562701824643e-09);
    q = fma(q, z, 1.6938509724371819e-06);
    q = fma(q, z, 2.3459619820224677e-04);
    q = fma(q, z, 2.1660849392498290e-02);
    q = fma(q, z, 1.0);
    q *= sh.pow32[n & 31];
    return __hiloint2double(__double2hiint(q) + ((n >> 5) << 20), __double2loint(q));
  };
  auto whole_of = [&](double w) __attribute__((always_inline)) {  // rounded to whole 2^-shift
    return (uint64_t)(__double_as_longlong(w + to_bits) - __double_as_longlong(to_bits));
  };

  // Kept: logits above `border`, and the first `ties` tokens that equal it, which weigh `tie` each.
  float border = -INFINITY;
  uint32_t ties = 0;
  double tie_w = 0.0;
  if (mx == INFINITY) {
    // it takes all: every +inf is a tie
    border = mx;
    tie_w = 1.0;
    uint32_t n = 0;
    each([&](float v) __attribute__((always_inline)) { n += v == mx; });
    n = (uint32_t)wave_sum_u64(n);
    if (lane == 0) sh.wave_cnt[wave] = n;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) ties += sh.wave_cnt[w];
    __syncthreads();
  }

  // f(logit, is one) with the logits above the border for which take(logit, index) holds, in no order:
  // as they stand where most are, else gathered
  auto each_kept = [&](auto take, auto f) __attribute__((always_inline)) {
    float* pend = &sh.pending[wave][0];
    int n = 0;
    each_vector([&](int i, const u32x4_t& vec) __attribute__((always_inline)) {
      uint64_t mask[EV];
      int more = 0;
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float v = smp_elem<BF16>(vec, e);
        mask[e] = __ballot(v > border && take(v, first + 64 * EV * i + e));
        more += (int)__popcll(mask[e]);
      }
      if (more > 32 * EV) {
#pragma unroll
        for (int e = 0; e < EV; ++e) f(smp_elem<BF16>(vec, e), (mask[e] >> lane) & 1);
        return true;
      }
      if (more == 0) return true;
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const int at = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask[e] >> 32),
                                                         __builtin_amdgcn_mbcnt_lo((uint32_t)mask[e], 0));
        if ((mask[e] >> lane) & 1) pend[at] = smp_elem<BF16>(vec, e);
        n += (int)__popcll(mask[e]);
      }
      asm volatile("" ::: "memory");  // a wave's LDS accesses are in order
      while (n >= 64 * SMP_GATHER) {
        n -= 64 * SMP_GATHER;
        float v[SMP_GATHER];
#pragma unroll
        for (int k = 0; k < SMP_GATHER; ++k) v[k] = pend[n + 64 * k + lane];
#pragma unroll
        for (int k = 0; k < SMP_GATHER; ++k) f(v[k], true);
      }
      asm volatile("" ::: "memory");
      return true;
    });
    for (; n > 0; n -= 64) f(pend[max(n - 64 + lane, 0)], n - 64 + lane >= 0);
  };
  auto all = [](float, int) { return true; };

  // Bins, even in the distance from the maximum, over what weighs anything; halves of the values, whose
  // difference cannot overflow.
  const float reach = min((float)((0.5 * mxd - 0.5 * (double)mn) * c), 0.5f * (float)(p.shift + 2));
  const float per =
      c > 0.0 && reach > 0.0f ? (float)min((double)(SMP_BINS - 1) / (double)reach * c, 3e38) : 0.0f;
  const float half_mx = 0.5f * mx;
  auto bin_of = [&](float v) __attribute__((always_inline)) {
    return (int)fminf(fmaf(-0.5f, v, half_mx) * per, (float)SMP_BINS);  // SMP_BINS: weighs nothing
  };

  double low = 0.0;  // min_p: lighter tokens are dropped; the largest logit always stays
  if (min_p > 0.0f) low = min((double)min_p, 1.0);
  // weight of what is kept: of all, of the waves before this one, and of this one
  uint64_t total = 0, before = 0, own = 0, tie_weight = 0;
  uint32_t ties_before = 0;
  bool summed = false;  // sh.wave_sum and sh.wave_cnt hold the waves' sums above the border, and their ties

  // The bin in which the sum of the bins reaches the goal, into sh.bin, what lies above it and up to its
  // end; goal: of the sum of all.
  auto scan_bins = [&](auto goal_of) __attribute__((always_inline)) {
    constexpr int EACH = SMP_BINS / TH;
    uint64_t mine[EACH], own_sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) own_sum += mine[i] = sh.bins[EACH * tid + i];
    uint64_t sum = wave_scan_u64(own_sum), sum_all = 0;
    if (lane == 63) sh.wave_sum[wave] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      sum += w < wave ? sh.wave_sum[w] : 0;
      sum_all += sh.wave_sum[w];
    }
    const uint64_t goal = goal_of(sum_all);
#pragma unroll
    for (int i = EACH - 1; i >= 0; --i) {
      if (sum >= goal && sum - mine[i] < goal) sh.bin = EACH * tid + i, sh.above = sum - mine[i], sh.upto = sum;
      sum -= mine[i];
    }
    __syncthreads();
    return goal;
  };
  // Where no bin has it: the goal lies among those that equal the old border, or nowhere.
  auto cut_ties = [&](uint64_t sum_all, uint64_t goal, uint64_t tie) __attribute__((always_inline)) {
    if (!tie || !ties) return;
    const uint64_t n = goal > sum_all ? (goal - sum_all + tie - 1) / tie : 0;
    if (n < ties) ties = (uint32_t)n;
  };
  // The border among the n tokens of the list, above which `above` lies.
  auto rank_list = [&](int n, uint64_t above, uint64_t goal, auto by_weight) __attribute__((always_inline)) {
    constexpr bool MASS = decltype(by_weight)::value;
    if (MASS) {
      for (int t = tid; t < n; t += TH) sh.weights[t] = whole_of(weight_of(sh.list[t]));
      __syncthreads();
    }
    for (int t = tid; t < n; t += TH) {
      const float v = sh.list[t];
      uint64_t more = above, same = 0;
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float o = sh.list[i];
        const uint64_t w = MASS ? sh.weights[i] : 1;
        more += o > v ? w : 0;
        same += o == v ? w : 0;
      }
      if (more < goal && goal <= more + same) {
        const uint64_t w = MASS ? sh.weights[t] : 1;
        sh.border = v;
        sh.ties = (uint32_t)((goal - more + w - 1) / w);
      }
    }
    __syncthreads();
    border = sh.border;
    ties = sh.ties;
    tie_w = weight_of(border);
  };
  // The same for a bin of more tokens, by halving the values: those above `lo` reach the goal, those
  // above `hi` do not.
  auto halve = [&](int at, uint64_t above, uint64_t goal, auto by_weight) __attribute__((always_inline)) {
    constexpr bool MASS = decltype(by_weight)::value;
    uint32_t lo = key_of(mn) - 1, hi = key_of(mx);
    uint64_t over = 0;  // weight of the bin's tokens above `hi`
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const float vm = logit_of(mid);
      uint64_t s = 0;
      each([&](float v) __attribute__((always_inline)) {
        if (v > vm && v > border && bin_of(v) == at) s += MASS ? whole_of(weight_of(v)) : 1;
      });
      s = wave_sum_u64(s);
      __syncthreads();
      if (lane == 0) sh.wave_sum[wave] = s;
      __syncthreads();
      s = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += sh.wave_sum[w];
      if (above + s >= goal) lo = mid;
      else hi = mid, over = s;
    }
    const float v = logit_of(hi);
    const uint64_t w = MASS ? whole_of(weight_of(v)) : 1;
    border = v;
    tie_w = weight_of(v);
    ties = (uint32_t)((goal - above - over + w - 1) / w);
  };
  auto clear = [&]() __attribute__((always_inline)) {
    for (int i = tid; i < SMP_BINS; i += TH) sh.bins[i] = 0;
    if (tid < WAVES) sh.wave_cnt[tid] = 0;
    if (tid == 0) sh.n_list = 0, sh.bin = SMP_BINS;
    __syncthreads();
  };

  // what lies above the border in the bins `from` to `at`, into the list
  auto gather = [&](int from, int at) __attribute__((always_inline)) {
    each_vector([&](int i, const u32x4_t& vec) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float v = smp_elem<BF16>(vec, e);
        const int b = bin_of(v);
        if (v > border && b >= from && b <= at) {
          const uint32_t k = atomicAdd(&sh.n_list, 1u);
          if (k < SMP_LIST) sh.list[k] = v, sh.index[k] = first + 64 * EV * i + e;
        }
      }
      return true;
    });
    __syncthreads();
    return (int)sh.n_list;
  };
  if (top_k > 0 && top_k < V) {
    int few = 0;  // tokens in the list, among them all that may be kept
    if (top_k <= SMP_FEW * 5 / 8) {
      // The top_k-th of the lanes' own maxima bounds the row's from below: a bin for each lane instead of
      // one for each token, and what lies above it is seldom much more than top_k tokens.
      clear();
      if (lane_mx > border && bin_of(lane_mx) < SMP_BINS) atomicAdd((uint32_t*)&sh.bins[bin_of(lane_mx)], 1u);
      __syncthreads();
      scan_bins([&](uint64_t) { return (uint64_t)top_k; });
      const int at = sh.bin;
      if (at < SMP_BINS) {
        few = gather(0, at);
        if (few > SMP_FEW) few = 0;
        __syncthreads();
      }
    }
    if (!few) {
      clear();
      each([&](float v) __attribute__((always_inline)) {
        const int b = bin_of(v);
        if (v > border && b < SMP_BINS) atomicAdd((uint32_t*)&sh.bins[b], 1u);
      });
      __syncthreads();
      uint64_t sum_all = 0;
      const uint64_t goal = scan_bins([&](uint64_t t) { sum_all = t; return (uint64_t)top_k; });
      const int at = sh.bin;
      if (at >= SMP_BINS) {
        cut_ties(sum_all, goal, 1);
      } else {
        const uint64_t above = sh.above, upto = sh.upto;
        const int n = gather(upto <= SMP_FEW ? 0 : at, at);
        if (upto <= SMP_FEW) few = n;
        else if (n > SMP_LIST) halve(at, above, goal, std::false_type{});
        else rank_list(n, above, goal, std::false_type{});
      }
      __syncthreads();
    }
    if (few) {
      // All in LDS: P threads for each token.  Its rank is how many keys lie below its own, of the logit
      // (from the largest) and the index; weights and indexes then stand in order of rank, in the bins.
      constexpr int P = TH / SMP_FEW, J = SMP_FEW / 64;
      uint64_t* key = sh.weights;
      uint64_t* w_at = sh.bins;
      int* i_at = (int*)(sh.bins + SMP_FEW);
      if (tid < few) key[tid] = (uint64_t)~key_of(sh.list[tid] + 0.0f) << 32 | (uint32_t)sh.index[tid];
      __syncthreads();
      const int mine = tid / P, m = min(few, top_k);
      if (mine < few) {
        const uint64_t own_key = key[mine];
        int r = 0;
#pragma unroll 4
        for (int i = tid % P; i < few; i += P) r += key[i] < own_key;
#pragma unroll
        for (int o = P / 2; o > 0; o >>= 1) r += __shfl_xor(r, o, 64);
        if (tid % P == 0) {
          const double w = weight_of(sh.list[mine]);
          w_at[r] = whole_of(w);
          i_at[r] = sh.index[mine];
          sh.pending[0][r] = w >= low ? 1.0f : 0.0f;
        }
      }
      __syncthreads();
      if (wave == 0) {
        // what lies before each one in order of rank; rank 64 j + lane
        uint64_t w[J], lies[J], sum_k = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          w[j] = lies[j] = 0;
          if (64 * j >= m) continue;
          w[j] = 64 * j + lane < m ? w_at[64 * j + lane] : 0;
          const uint64_t to = wave_scan_u64(w[j]);
          lies[j] = sum_k + to - w[j];
          sum_k += __shfl(to, 63, 64);
        }
        uint64_t goal_p = sum_k;
        if (top_p < 1.0f) {
          const double share = ceil((double)top_p * (double)sum_k);
          goal_p = share >= 1.0 ? (uint64_t)share : 1;
        }
        uint64_t kept = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (64 * j + lane >= m) continue;
          if (!(lies[j] < goal_p && sh.pending[0][64 * j + lane] != 0.0f)) w[j] = 0;
          kept += w[j];
          w_at[64 * j + lane] = w[j];
        }
        kept = wave_sum_u64(kept);
        if (lane == 0) sh.above = kept;
      }
      __syncthreads();
      total = sh.above;
      const double t = (double)u * (double)total;
      uint64_t target = t > 0.0 ? (uint64_t)t : 0;
      if (target >= total) target = total - 1;
      if (mine < m) {
        const int idx = i_at[mine];
        const uint64_t w = w_at[mine];
        uint64_t ahead = 0;  // what lies before it in order of index
#pragma unroll 4
        for (int i = tid % P; i < m; i += P) ahead += i_at[i] < idx ? w_at[i] : 0;
#pragma unroll
        for (int o = P / 2; o > 0; o >>= 1) ahead += __shfl_xor(ahead, o, 64);
        if (tid % P == 0 && w && ahead <= target && target < ahead + w) {
          p.tokens[row] = idx;
          if (p.probs) p.probs[row] = (float)((double)w / (double)total);
        }
      }
      return;
    }
  }
  if (top_p < 1.0f) {
    clear();
    each_kept(all, [&](float v, bool is) __attribute__((always_inline)) {
      const int b = bin_of(v);
      const uint64_t w = whole_of(weight_of(v));
      if (is && b < SMP_BINS) atomicAdd((unsigned long long*)&sh.bins[b], (unsigned long long)w);
    });
    __syncthreads();
    const uint64_t tie = ties ? whole_of(tie_w) : 0;
    uint64_t sum_all = 0;
    const uint64_t goal = scan_bins([&](uint64_t t) {
      sum_all = t;
      const double share = ceil((double)top_p * (double)(t + ties * tie));
      return share >= 1.0 ? (uint64_t)share : (uint64_t)1;
    });
    const int at = sh.bin;
    const uint64_t above = sh.above;
    if (at >= SMP_BINS) {
      cut_ties(sum_all, goal, tie);
    } else {
      // the border's bin goes to the list; what lies above it is kept, and summed on the way
      uint64_t m = 0;
      each_kept(
          [&](float v, int idx) __attribute__((always_inline)) {
            const int b = bin_of(v);
            if (b == at) {
              const uint32_t k = atomicAdd(&sh.n_list, 1u);
              if (k < SMP_LIST) sh.list[k] = v, sh.index[k] = idx;
            }
            return b < at;
          },
          [&](float v, bool is) __attribute__((always_inline)) {
            const double w = weight_of(v);
            const uint64_t whole = whole_of(w);
            m += is && w >= low ? whole : 0;
          });
      m = wave_sum_u64(m);
      __syncthreads();
      const int n = (int)sh.n_list;
      if (n <= SMP_LIST) {
        rank_list(n, above, goal, std::true_type{});
        if (lane == 0) sh.wave_sum[wave] = m;
        __syncthreads();
        for (int t = tid; t < n; t += TH) {
          const float v = sh.list[t];
          const int w = sh.index[t] / (layers * 64 * EV);
          if (v > border && weight_of(v) >= low)
            atomicAdd((unsigned long long*)&sh.wave_sum[w], (unsigned long long)sh.weights[t]);
          if (v == border) atomicAdd(&sh.wave_cnt[w], 1u);
        }
        summed = true;
      } else {
        halve(at, above, goal, std::true_type{});
      }
    }
    __syncthreads();
  }
  if (!summed) {
    uint64_t m = 0;
    uint32_t n = 0;
    each_kept(all, [&](float v, bool is) __attribute__((always_inline)) {
      const double w = weight_of(v);
      const uint64_t whole = whole_of(w);
      m += is && w >= low ? whole : 0;
    });
    if (ties) each([&](float v) __attribute__((always_inline)) { n += v == border; });
    m = wave_sum_u64(m);
    n = (uint32_t)wave_sum_u64(n);
    if (lane == 0) sh.wave_sum[wave] = m, sh.wave_cnt[wave] = n;
    __syncthreads();
  }
  tie_weight = ties && tie_w >= low ? whole_of(tie_w) : 0;
  {
    uint32_t seen = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) before = total, ties_before = seen;
      const uint32_t left = ties > seen ? ties - seen : 0;
      const uint64_t of_wave = sh.wave_sum[w] + tie_weight * min(left, sh.wave_cnt[w]);
      if (w == wave) own = of_wave;
      total += of_wave;
      seen += sh.wave_cnt[w];
    }
  }

  // the token at which the kept weight passes u * total
  const double t = (double)u * (double)total;
  uint64_t target = t > 0.0 ? (uint64_t)t : 0;
  if (target >= total) target = total - 1;
  if (target < before || target - before >= own) return;
  uint64_t acc = before;
  uint32_t seen = ties_before;
  each_vector([&](int i, const u32x4_t& vec) __attribute__((always_inline)) {
    // ties of the lanes before this one
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < EV; ++e) n += smp_elem<BF16>(vec, e) == border;
    uint32_t rank = seen, all_ties = 0;
    if (__any(n)) {
      const uint32_t upto = (uint32_t)wave_scan_u64(n);
      rank += upto - n;
      all_ties = (uint32_t)__shfl((int)upto, 63, 64);
    }
    uint64_t m = 0, w[EV];
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      const float v = smp_elem<BF16>(vec, e);
      w[e] = 0;
      if (v > border) {
        const double d = weight_of(v);
        w[e] = d >= low ? whole_of(d) : 0;
      } else if (v == border) {
        w[e] = rank < ties ? tie_weight : 0;
        ++rank;
      }
      m += w[e];
    }
    const uint64_t upto = acc + wave_scan_u64(m), from = upto - m;
    if (from <= target && target < upto) {
      uint64_t s = from;
      bool open = true;
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        s += w[e];
        if (open && s > target) {
          open = false;
          p.tokens[row] = first + 64 * EV * i + e;
          if (p.probs) p.probs[row] = (float)((double)w[e] / (double)total);
        }
      }
    }
    acc = __shfl(upto, 63, 64);
    seen += all_ties;
    return acc <= target;
  });
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" int mi_sample(void* stream, const void* logits, int32_t dtype, int64_t ld, int64_t rows, int64_t vocab,
                         const mi_sampling* how, const float* u, int32_t* tokens, float* probs) {
  if (rows < 0 || vocab < 0) return host_fail(MI_ERR_SHAPE, "negative size");
  if (dtype != MI_F32 && dtype != MI_BF16) return host_fail(MI_ERR_DTYPE, "dtype %d", dtype);
  if (rows == 0) return MI_OK;
  if (vocab == 0) return host_fail(MI_ERR_SHAPE, "vocab is 0: there is no token to pick");
  if (rows > INT32_MAX || vocab > (1 << 24))
    return host_fail(MI_ERR_SHAPE, "rows=%lld exceeds 2^31-1 or vocab=%lld exceeds 2^24", (long long)rows,
                     (long long)vocab);
  if (!logits || !how || !u || !tokens) return host_fail(MI_ERR_NULL, "logits, how, u or tokens is NULL");
  if (rows > 1 && ld < vocab)
    return host_fail(MI_ERR_LD, "ld=%lld < vocab=%lld", (long long)ld, (long long)vocab);
  if ((uintptr_t)logits % (dtype == MI_BF16 ? 2 : 4) || ((uintptr_t)u & 3) || ((uintptr_t)tokens & 3) ||
      ((uintptr_t)probs & 3) || ((uintptr_t)how->temperature & 3) || ((uintptr_t)how->top_k & 3) ||
      ((uintptr_t)how->top_p & 3) || ((uintptr_t)how->min_p & 3))
    return host_fail(MI_ERR_UNSUPPORTED, "pointers must be aligned to their element size");
  const int st = host_device();
  if (st != MI_OK) return st;
  SampleParams p;
  p.logits = logits;
  p.ld = ld;
  p.vocab = (int)vocab;
  int bits = 0;
  while ((int64_t{1} << bits) < vocab) ++bits;
  p.shift = 62 - bits < 50 ? 62 - bits : 50;
  p.u = u;
  p.tokens = tokens;
  p.probs = probs;
  p.how = *how;
  const bool bf16 = dtype == MI_BF16;
  // More rows than CUs: half the threads, so that two rows share a CU and one's waits are under the
  // other's work (512 rows of 32000 bf16 logits, top-p: 65 us with 1024 threads, 60 with 512)
  const int threads = rows > host_cus() ? 512 : 1024;
  const int per_layer = threads * (bf16 ? 8 : 4);
  p.layers = (int)((vocab + per_layer - 1) / per_layer);
  const bool aligned = ((uintptr_t)logits & 15) == 0 && (rows == 1 || ld % (bf16 ? 8 : 4) == 0);
  auto kernel = sample_kernel<1024, true, true>;
  if (threads == 1024)
    kernel = bf16 ? (aligned ? sample_kernel<1024, true, true> : sample_kernel<1024, true, false>)
                  : (aligned ? sample_kernel<1024, false, true> : sample_kernel<1024, false, false>);
  else
    kernel = bf16 ? (aligned ? sample_kernel<512, true, true> : sample_kernel<512, true, false>)
                  : (aligned ? sample_kernel<512, false, true> : sample_kernel<512, false, false>);
  kernel<<<(unsigned)rows, threads, 0, (hipStream_t)stream>>>(p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "sample launch: %s", hipGetErrorString(e));
}
