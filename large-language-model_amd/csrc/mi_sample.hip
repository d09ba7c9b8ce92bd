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
// The largest top-k that the lanes' maxima are asked for.  Their bound lets a few dozen tokens more than top-k through,
// and where those do not fit the list the histogram follows all the same.  With 0 / 160 / 255 here (us, top-p 0.9):
//    rows of logits           top-k 50        160             180             200             220
//      64 of 32001, fp32      16.0/12.8/12.8  19.5/16.5/16.5  19.9/20.2/17.1  21.1/21.4/18.3  21.7/22.0/27.6
//     512 of 32000, fp32      34.1/25.8/25.7  39.4/31.6/31.6  40.5/40.9/33.2  41.7/42.1/47.3  42.7/43.2/52.5
//      64 of 5000, fp32       10.4/9.7/9.7    13.5/12.9/13.0  14.0/14.2/13.5  15.2/15.5/14.8  15.7/16.0/19.4
constexpr int SMP_FEW_K = SMP_FEW * 5 / 8;
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

// 16 bytes at any element: odd pitches and vocabularies put rows anywhere, and one such load takes less
// than eight (64 rows of 50257 bf16 logits, top-p: 36 us against 57; where aligned, the same).
typedef uint32_t u32x4_any_t __attribute__((ext_vector_type(4), aligned(2)));

// Elements j .. of a row of V as one vector; past the row's end -inf.
template <bool BF16>
__device__ __forceinline__ u32x4_t smp_load(const void* row, int j, int V) {
  constexpr int EV = BF16 ? 8 : 4;
  const uint32_t none = BF16 ? 0xff80ff80u : 0xff800000u;
  u32x4_t v = {none, none, none, none};
  if (j + EV <= V) return *(const u32x4_any_t*)((const char*)row + (int64_t)j * (BF16 ? 2 : 4));
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

// The vectors of this lane of a row of V: vector i of a wave's run of `layers` holds the elements from
// first + 64 EV i on.  ahead() only asks for one, without a branch, so that the wait for those asked for
// before need not be for this one too; at() is what it holds, which past the row's end is read again there.
__device__ const uint32_t smp_none[4] = {0, 0, 0, 0};
template <bool BF16>
struct SampleRun {
  static constexpr int EV = BF16 ? 8 : 4;
  const char* row;
  int V, first, wave_first;
  __device__ __forceinline__ SampleRun(const SampleParams& p, int r)
      : row((const char*)p.logits + (int64_t)r * p.ld * (BF16 ? 2 : 4)), V(p.vocab) {
    wave_first = uniform(threadIdx.x >> 6) * p.layers * 64 * EV;
    first = wave_first + (int)(threadIdx.x & 63) * EV;
  }
  __device__ __forceinline__ u32x4_t ahead(int i) const {
    const char* at = row + (int64_t)min(first + 64 * EV * i, V - EV) * (BF16 ? 2 : 4);
    return *(const u32x4_any_t*)(V >= EV ? at : (const char*)smp_none);
  }
  __device__ __forceinline__ u32x4_t at(u32x4_t v, int i) const {
    if (wave_first + 64 * EV * (i + 1) > V) {
      v = smp_load<BF16>(row, first + 64 * EV * i, V);
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), here and not where the branches meet
    }
    return v;
  }
};

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

// Weights of logits up to a finite maximum.
struct SampleWeights {
  double mx, c32, to_bits;  // w + to_bits: w * 2^shift, rounded, in the low bits
  const double* pow32;      // LDS, 2^(j/32)
  __device__ __forceinline__ SampleWeights(float mx_, float T, int shift, const double* pow32_)
      : mx((double)mx_), c32(32.0 * (1.4426950408889634074 / (double)T)),
        to_bits(1.5 * (double)(uint64_t{1} << (52 - shift))), pow32(pow32_) {}
  __device__ __forceinline__ double of(float v) const {  // as a 64-bit float
    const double y = max(((double)v - mx) * c32, -2048.0);  // 32 y; 2^-64 rounds to nothing
    const double t = y + 6755399441055744.0;                // 1.5 * 2^52: rounded, in the low bits
    const int n = (int)(uint32_t)__double_as_longlong(t);
    const double z = y - (t - 6755399441055744.0);          // |z| <= 1/2, of 1/32
    // 2^(z/32) = sum (z ln 2 / 32)^k / k!, past k = 5 below 2^-48
    double q = 3.9737099845494154e-11;
    q = fma(q, z, 9.172562701824643e-09);
    q = fma(q, z, 1.6938509724371819e-06);
    q = fma(q, z, 2.3459619820224677e-04);
    q = fma(q, z, 2.1660849392498290e-02);
    q = fma(q, z, 1.0);
    q *= pow32[n & 31];
    return __hiloint2double(__double2hiint(q) + ((n >> 5) << 20), __double2loint(q));
  }
  __device__ __forceinline__ uint64_t whole(double w) const {  // rounded to whole 2^-shift
    return (uint64_t)(__double_as_longlong(w + to_bits) - __double_as_longlong(to_bits));
  }
};

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

template <int TH, bool BF16>
__device__ __forceinline__ void sample_row(const SampleParams& p, int row, SampleShared<TH / 64>& sh) {
  constexpr int EV = BF16 ? 8 : 4, WAVES = TH / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int V = p.vocab, layers = p.layers;
  // a whole number of layers covers the row, so runs of the last waves may lie past its end (the sum
  // stays below 2^25)
  const SampleRun<BF16> run(p, row);
  const int first = run.first;
  // f(i, vector) over this lane's vectors, the next one on its way; f returns whether to go on (the
  // same in all lanes)
  auto each_vector = [&](auto f) __attribute__((always_inline)) {
    u32x4_t v = run.ahead(0);
    for (int i = 0; i < layers; ++i) {
      const u32x4_t next = run.ahead(i + 1);
      if (!f(i, run.at(v, i))) break;
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
  for (int i0 = 0; i0 < layers; i0 += 4) {  // four vectors on their way: this pass waits for memory
    u32x4_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = run.ahead(i0 + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j >= layers) break;
      const u32x4_t vec = run.at(v[j], i0 + j);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        const float l = smp_elem<BF16>(vec, e);
        mx = fmaxf(mx, l);
        mn = fminf(mn, l > -INFINITY ? l : INFINITY);
      }
    }
  }
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

  const SampleWeights W(mx, T, p.shift, sh.pow32);
  const double c = W.c32 * 0.03125, mxd = W.mx;
  auto weight_of = [&](float v) __attribute__((always_inline)) { return W.of(v); };
  auto whole_of = [&](double w) __attribute__((always_inline)) { return W.whole(w); };

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
  // difference cannot overflow.  64 bits until the division: with a temperature of 1e38 a reach in 32 is a
  // denormal of few bits, and the row's tail would lie past the last bin.
  const double reach = min((0.5 * mxd - 0.5 * (double)mn) * c, 0.5 * (double)(p.shift + 2));
  const float per = c > 0.0 && reach > 0.0 ? (float)min((double)(SMP_BINS - 1) / reach * c, 3e38) : 0.0f;
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
    if (top_k <= SMP_FEW_K) {
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
    auto weigh = [&](float v, bool is) __attribute__((always_inline)) {
      const int b = bin_of(v);
      const uint64_t w = whole_of(weight_of(v));
      if (is && b < SMP_BINS) atomicAdd((unsigned long long*)&sh.bins[b], (unsigned long long)w);
    };
    if (border == -INFINITY) {
      // a vector's weights side by side: the asm keeps them out of the branches about the sums
      each_vector([&](int, const u32x4_t& vec) __attribute__((always_inline)) {
        uint64_t w[EV];
#pragma unroll
        for (int e = 0; e < EV; ++e) w[e] = whole_of(weight_of(smp_elem<BF16>(vec, e)));
#pragma unroll
        for (int e = 0; e < EV; ++e) asm volatile("" : "+v"(w[e]));
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const int b = bin_of(smp_elem<BF16>(vec, e));  // SMP_BINS of -inf and NaN
          if (b < SMP_BINS) atomicAdd((unsigned long long*)&sh.bins[b], (unsigned long long)w[e]);
        }
        return true;
      });
    } else {
      each_kept(all, weigh);
    }
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

template <int TH, bool BF16>
__global__ void __launch_bounds__(TH) sample_kernel(SampleParams p) {
  __shared__ SampleShared<TH / 64> sh;
  sample_row<TH, BF16>(p, blockIdx.x, sh);
}

// Long rows of bf16 logits hold few distinct ones (32000 normal ones about 2200): they are counted by
// their bits, 32768 counters of 16 bits in LDS, and listed in order with their counts, so only the
// distinct ones are weighed and all three borders lie in running sums over the list.  The second pass
// takes each token's weight from LDS by its bits.  The answers are those of the kernel above, to the bit.
// Normal logits of standard deviation 2.5, top-p 0.9, without / with it (us):
//             4096       8192       16384      32000      131072 logits
//    64 rows  13.9/14.7  15.0/15.3  20.7/18.1  33.3/23.4  102/59
//   512 rows  15.1/17.1  20.9/19.9  31.6/25.6  54.8/39.2  213/117
// Where a row is so flat that more distinct logits are kept than there is room for weights, it takes both: 64 rows of
// 32000 with top-p 0.9, deviations of 0.5, 1, 1.5 and 4: 36.2/48.2, 36.6/47.6, 35.6/23.6, 28.8/23.4; with top-p 0.99, 1,
// 2 and 2.5: 35.3/46.7, 36.5/47.8, 35.3/23.6.
// LDS and vector instructions bound it: of a row's 17 us alone 4 go to the counting, 4 to the second
// pass, 7 to the list and its sums.  80 KB of LDS leave room for two blocks of 512 threads on a CU.
constexpr int SMC_LIST = 3584;          // distinct logits of a row
constexpr int SMC_KEPT = SMC_LIST / 2;  // of them above the border: their 64-bit weights fill the list
constexpr int SMC_FROM = 8192;          // logits of a row from which it pays to clear and read the counters

template <int WAVES>
struct SampleCounts {
  uint32_t count[16384];  // two 16-bit counters each; then the kept logits' places in the list
  union {
    uint32_t list[SMC_LIST];     // place << 16 | count, from the largest
    uint64_t weights[SMC_KEPT];  // of the kept ones
  };
  uint16_t chunk[256] __attribute__((aligned(16)));  // distinct logits of 128 places
  double pow32[32];
  uint64_t wave_sum[WAVES];
  uint32_t wave_cnt[WAVES];
  uint64_t above, weight;
  uint32_t entry, place, ties, other;
};

// Finite logits have places in order if they are 0 or their absolute value lies in [2^-64, 2^64), the
// uppermost two of that left out: zeros 0x4000, the others from there by their absolute bits.  -inf has
// one below 0; the rest (`other`) is left to the general kernel.
constexpr int SMC_ZERO = 0x4000, SMC_FIRST = 63 << 7;  // exponent -64
__device__ __forceinline__ int place_of(uint32_t h) {
  const int a = (int)(h & 0x7fffu), d = a ? a - (SMC_FIRST - 1) : 0;
  return SMC_ZERO + ((h & 0x8000u) ? -d : d);
}
__device__ __forceinline__ bool has_place(uint32_t h) {
  const uint32_t a = h & 0x7fffu;
  return a == 0 || a - SMC_FIRST < (uint32_t)SMC_ZERO - 1;
}
// The places of two logits at once, of those that have one; -inf below all of them.
typedef int16_t s16x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ s16x2_t places_of(uint32_t hh) {
  const s16x2_t a = __builtin_bit_cast(s16x2_t, hh & 0x7fff7fffu), sign = __builtin_bit_cast(s16x2_t, hh) >> 15;
  const s16x2_t d = __builtin_elementwise_max(a - (int16_t)(SMC_FIRST - 1), s16x2_t{0, 0});
  return (d ^ sign) - sign + (int16_t)SMC_ZERO;
}
__device__ __forceinline__ float logit_at(int place) {
  const int d = place - SMC_ZERO, a = abs(d) + SMC_FIRST - 1;
  return d == 0 ? 0.0f : bf16_bits_to_f32((uint32_t)(d < 0 ? a | 0x8000 : a));
}

// How many bits of a wave's mask belong to lanes before this one.
__device__ __forceinline__ uint32_t lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Whether it has answered; if not (a logit without a place, too many distinct ones or
// too many alike) nothing is written.
template <int TH>
__device__ __forceinline__ bool sample_counted(const SampleParams& p, int row, float T, int top_k, float top_p,
                                               float min_p, SampleCounts<TH / 64>& sh) {
  constexpr int EV = 8, WAVES = TH / 64, EACH = (SMC_LIST + TH - 1) / TH;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), V = p.vocab, layers = p.layers;
  const SampleRun<true> run(p, row);
  const int first = run.first;
  // four vectors are under way at a time
  u32x4_t vec[4];
  auto fetch = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) vec[j] = smp_load<true>(run.row, first + 64 * EV * (i0 + j), V);
  };
  auto each_vector = [&](auto f) __attribute__((always_inline)) {
    for (int i0 = 0; i0 < layers; i0 += 4) {
      if (i0) fetch(i0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j < layers && !f(i0 + j, vec[j])) return;
    }
  };
  auto bits_at = [&](const u32x4_t& v, int e) { return (e & 1) ? v[e >> 1] >> 16 : v[e >> 1] & 0xffffu; };
  fetch(0);
#pragma unroll
  for (int i = 0; i < 4096 / TH; ++i) *(u32x4_t*)(sh.count + 4 * (tid + TH * i)) = u32x4_t{0, 0, 0, 0};
  if (tid < 32) sh.pow32[tid] = exp2(tid * 0.03125);
  if (tid == 0) sh.other = 0;
  __syncthreads();
  uint32_t finite = 0;
  each_vector([&](int, const u32x4_t& v) __attribute__((always_inline)) {
    // the largest and the least absolute bits, zeros aside
    u16x2_t most = {0, 0}, least = {0xffff, 0xffff};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u16x2_t a = __builtin_bit_cast(u16x2_t, v[i] & 0x7fff7fffu);
      most = __builtin_elementwise_max(most, a);
      least = __builtin_elementwise_min(least, (u16x2_t)(a - (uint16_t)1));
    }
    if (max(most.x, most.y) >= SMC_FIRST + SMC_ZERO - 1 || min(least.x, least.y) < SMC_FIRST - 1) {
#pragma unroll
      for (int e = 0; e < EV; ++e)
        if (!has_place(bits_at(v, e)) && bits_at(v, e) != 0xff80u) sh.other = 1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const s16x2_t at = places_of(v[i]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int k = e ? at.y : at.x;  // below 0: -inf, or too large
        finite += k >= 0;
        if (k >= 0) atomicAdd(&sh.count[k >> 1], 1u << ((k & 1) << 4));
      }
    }
    return true;
  });
  finite = (uint32_t)wave_sum_u64(finite);
  if (lane == 0) sh.wave_cnt[wave] = finite;
  __syncthreads();
  finite = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) finite += sh.wave_cnt[i];

  // The list, from the largest down: 256 chunks of 128 places, dealt to the waves in turn, since most
  // of them are empty and the others lie together.
  constexpr int CHUNKS = 16384 / 64, STEPS = CHUNKS / WAVES, GROUPS = WAVES / 4;
  const int word0 = 16383 - wave * 64 - lane;  // of the wave's first chunk
#pragma unroll 8
  for (int i = 0; i < STEPS; ++i) {
    const uint32_t w = sh.count[word0 - 64 * WAVES * i];
    const uint32_t n = __popcll(__ballot(w & 0xffffu)) + __popcll(__ballot(w >> 16));
    if (lane == 0) sh.chunk[WAVES * i + wave] = (uint16_t)n;
  }
  __syncthreads();
  if (sh.other) return false;
  uint32_t n_list;
  {
    // lane l adds up the chunks 4 l .. 4 l + 3; the wave's own are with the lanes GROUPS i + wave / 4
    const u32x2_t c = *(const u32x2_t*)(sh.chunk + 4 * lane);
    uint32_t sum = 0, before = 0, own = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t n = (e & 1) ? c[e >> 1] >> 16 : c[e >> 1] & 0xffffu;
      if (e == wave % 4) before = sum, own = n;
      sum += n;
    }
    const uint32_t to = (uint32_t)wave_scan_u64(sum);
    before += to - sum;
    n_list = (uint32_t)__builtin_amdgcn_readlane((int)to, 63);
    if (finite == 0) {
      if (tid == 0) {
        p.tokens[row] = -1;
        if (p.probs) p.probs[row] = 0.0f;
      }
      return true;
    }
    if (n_list == 0 || n_list > SMC_LIST) return false;
    uint64_t full = __ballot(own && lane % GROUPS == wave / 4);
    while (full) {
      const int l = __ffsll((unsigned long long)full) - 1;
      full &= full - 1;
      const int word = word0 - 64 * WAVES * (l / GROUPS);
      const uint32_t w = sh.count[word];
      uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)before, l) + lanes_below(__ballot(w & 0xffffu)) +
                    lanes_below(__ballot(w >> 16));
      if (w >> 16) sh.list[at++] = (uint32_t)(2 * word + 1) << 16 | w >> 16;
      if (w & 0xffffu) sh.list[at] = (uint32_t)(2 * word) << 16 | (w & 0xffffu);
    }
  }
  __syncthreads();
  const SampleWeights W(logit_at(sh.list[0] >> 16), T, p.shift, sh.pow32);

  // Entries each * tid .., their weights, and running sums of tokens and weight.
  const int each = (int)(n_list + TH - 1) / TH;
  uint32_t place[EACH], n[EACH];
  uint64_t w[EACH], mass = 0;
  uint32_t tokens = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = each * tid + i;
    place[i] = n[i] = 0;
    w[i] = 0;
    if (i < each && e < (int)n_list) {
      const uint32_t v = sh.list[e];
      place[i] = v >> 16;
      n[i] = v & 0xffffu;
      w[i] = W.whole(W.of(logit_at(place[i])));
    }
    tokens += n[i];
    mass += n[i] * w[i];
  }
  const uint64_t mass_to = wave_scan_u64(mass);
  const uint32_t tokens_to = (uint32_t)wave_scan_u64(tokens);
  if (lane == 63) sh.wave_sum[wave] = mass_to, sh.wave_cnt[wave] = tokens_to;
  __syncthreads();
  uint64_t mass0 = mass_to - mass, total = 0;  // before this thread's entries
  uint32_t tokens0 = tokens_to - tokens, all_tokens = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    mass0 += i < wave ? sh.wave_sum[i] : 0;
    tokens0 += i < wave ? sh.wave_cnt[i] : 0;
    total += sh.wave_sum[i];
    all_tokens += sh.wave_cnt[i];
  }
  // A counter that ran over has lost 65536 tokens, and may have given its neighbour one.
  if (all_tokens != finite) return false;
  // Kept: entries before `entry`, and the first `ties` tokens of it.
  uint32_t entry = n_list - 1, ties = sh.list[n_list - 1] & 0xffffu;
  if (top_k > 0 && (uint32_t)top_k < all_tokens) {
    uint32_t t = tokens0;
    uint64_t m = mass0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (t < (uint32_t)top_k && (uint32_t)top_k <= t + n[i]) {
        sh.entry = each * tid + i;
        sh.ties = top_k - t;
        sh.above = m + (top_k - t) * w[i];
      }
      t += n[i];
      m += n[i] * w[i];
    }
    __syncthreads();
    entry = sh.entry;
    ties = sh.ties;
    total = sh.above;
    __syncthreads();
  }
  if (top_p < 1.0f) {
    const double share = ceil((double)top_p * (double)total);
    const uint64_t goal = share >= 1.0 ? (uint64_t)share : 1;
    uint64_t m = mass0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const uint64_t to = m + n[i] * w[i];
      if (m < goal && goal <= to) {
        sh.entry = each * tid + i;
        sh.ties = (uint32_t)((goal - m + w[i] - 1) / w[i]);
      }
      m = to;
    }
    __syncthreads();
    if (sh.entry < entry) entry = sh.entry, ties = sh.ties;
    else if (sh.entry == entry) ties = min(ties, sh.ties);
    __syncthreads();
  }
  if (min_p > 0.0f) {
    // the last entry that weighs enough; the first always does
    const double low = min((double)min_p, 1.0);
    if (tid == 0) sh.entry = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (n[i] && (uint32_t)(each * tid + i) <= entry && W.of(logit_at(place[i])) >= low)
        atomicMax(&sh.entry, (uint32_t)(each * tid + i));
    __syncthreads();
    if (sh.entry < entry) entry = sh.entry, ties = sh.list[entry] & 0xffffu;
  }
  if (entry >= SMC_KEPT) return false;
  __syncthreads();  // the list has been read
  {
    uint64_t m = mass0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const uint32_t e = each * tid + i;
      if (n[i] && e < entry) {
        sh.weights[e] = w[i];
        ((uint16_t*)sh.count)[place[i]] = (uint16_t)e;
      } else if (n[i] && e == entry) {
        sh.weights[e] = 0;  // its tokens count by their order
        ((uint16_t*)sh.count)[place[i]] = (uint16_t)e;
        sh.place = place[i];
        sh.weight = w[i];
        sh.above = m + ties * w[i];
      }
      m += n[i] * w[i];
    }
  }
  __syncthreads();
  const int border = sh.place;
  const uint64_t tie_weight = sh.weight;
  total = sh.above;

  // Each wave's weight above the border, and its ties.
  auto weight_at = [&](int at) __attribute__((always_inline)) {
    return sh.weights[((const uint16_t*)sh.count)[max(at, border)]];
  };
  fetch(0);
  uint64_t m = 0;
  uint32_t nt = 0;
  const s16x2_t borders = {(int16_t)border, (int16_t)border};
  each_vector([&](int, const u32x4_t& v) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const s16x2_t k = places_of(v[i]), at = __builtin_elementwise_max(k, borders);
      m += sh.weights[((const uint16_t*)sh.count)[at.x]] + sh.weights[((const uint16_t*)sh.count)[at.y]];
      nt += (k.x == border) + (k.y == border);
    }
    return true;
  });
  m = wave_sum_u64(m);
  nt = (uint32_t)wave_sum_u64(nt);
  if (lane == 0) sh.wave_sum[wave] = m, sh.wave_cnt[wave] = nt;
  __syncthreads();
  uint64_t acc = 0, own = 0, sum = 0;
  uint32_t seen = 0, all_seen = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    if (i == wave) acc = sum, seen = all_seen;
    const uint32_t left = ties > all_seen ? ties - all_seen : 0;
    const uint64_t of_wave = sh.wave_sum[i] + tie_weight * min(left, sh.wave_cnt[i]);
    if (i == wave) own = of_wave;
    sum += of_wave;
    all_seen += sh.wave_cnt[i];
  }
  const double t = (double)p.u[row] * (double)total;
  uint64_t target = t > 0.0 ? (uint64_t)t : 0;
  if (target >= total) target = total - 1;
  if (target < acc || target - acc >= own) return true;
  if (layers > 4) fetch(0);
  each_vector([&](int i, const u32x4_t& v) __attribute__((always_inline)) {
    uint32_t ties_here = 0;
#pragma unroll
    for (int e = 0; e < EV; ++e) ties_here += place_of(bits_at(v, e)) == border;
    uint32_t rank = seen, all_ties = 0;
    if (__any(ties_here)) {
      const uint32_t upto = (uint32_t)wave_scan_u64(ties_here);
      rank += upto - ties_here;
      all_ties = (uint32_t)__shfl((int)upto, 63, 64);
    }
    uint64_t we[EV], s = 0;
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      const int k = place_of(bits_at(v, e));
      we[e] = k == border && rank < ties ? tie_weight : weight_at(k);
      rank += k == border;
      s += we[e];
    }
    const uint64_t upto = acc + wave_scan_u64(s), from = upto - s;
    if (from <= target && target < upto) {
      uint64_t run = from;
      bool open = true;
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        run += we[e];
        if (open && run > target) {
          open = false;
          p.tokens[row] = first + 64 * EV * i + e;
          if (p.probs) p.probs[row] = (float)((double)we[e] / (double)total);
        }
      }
    }
    acc = __shfl(upto, 63, 64);
    seen += all_ties;
    return acc <= target;
  });
  return true;
}

// Whether a border is looked for among many tokens.  (64 rows of 32000, without counts and with: top-k 200 21.0 and
// 22.6 us, 260 24.9 and 22.6, 1000 26.6 and 23.1; min-p alone 19.5 and 29.1.)
__host__ __device__ __forceinline__ bool counts_pay(int top_k, float top_p, int vocab) {
  return top_k > 0 && top_k < vocab ? top_k > SMP_FEW : top_p < 1.0f;
}

// Long rows of bf16 logits.
template <int TH>
__global__ void __launch_bounds__(TH) sample_counts_kernel(SampleParams p) {
  __shared__ union {
    SampleCounts<TH / 64> counted;
    SampleShared<TH / 64> general;
  } sh;
  const int row = blockIdx.x;
  const float T = p.how.temperature ? p.how.temperature[row] : p.how.temperature_all;
  const int top_k = p.how.top_k ? p.how.top_k[row] : p.how.top_k_all;
  const float top_p = p.how.top_p ? p.how.top_p[row] : p.how.top_p_all;
  const float min_p = p.how.min_p ? p.how.min_p[row] : p.how.min_p_all;
  if (T > 0.0f && counts_pay(top_k, top_p, p.vocab)) {
    if (sample_counted<TH>(p, row, T, top_k, top_p, min_p, sh.counted)) return;
    __syncthreads();
  }
  sample_row<TH, true>(p, row, sh.general);
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
  if (rows > 1 && ld != 0 && ld < vocab)
    return host_fail(MI_ERR_LD, "ld=%lld < vocab=%lld", (long long)ld, (long long)vocab);
  if ((uintptr_t)logits % (dtype == MI_BF16 ? 2 : 4) || ((uintptr_t)u & 3) || ((uintptr_t)tokens & 3) ||
      ((uintptr_t)probs & 3) || ((uintptr_t)how->temperature & 3) || ((uintptr_t)how->top_k & 3) ||
      ((uintptr_t)how->top_p & 3) || ((uintptr_t)how->min_p & 3))
    return host_fail(MI_ERR_UNSUPPORTED, "pointers must be aligned to their element size");
  const int st = host_device();
  if (st != MI_OK) return st;
  SampleParams p;
  p.ld = ld;
  p.vocab = (int)vocab;
  int bits = 0;
  while ((int64_t{1} << bits) < vocab) ++bits;
  p.shift = 62 - bits < 50 ? 62 - bits : 50;
  const bool bf16 = dtype == MI_BF16;
  // Whether any row may gain by counts; each decides for itself.
  const bool counted = bf16 && vocab >= SMC_FROM &&
                       (how->temperature || how->temperature_all > 0.0f) &&
                       (how->top_k || how->top_p || counts_pay(how->top_k_all, how->top_p_all, (int)vocab));
  // More rows than CUs: half the threads, so that two rows share a CU and one's waits are under the
  // other's work (bf16 rows of 32000, top-p, by weights, with 1024 / 512 threads: 256 rows 37.6/44.4 us, 257
  // 65.0/54.4, 512 72.7/63.3)
  const bool halved = rows > host_cus();
  const int threads = halved ? 512 : 1024, per_layer = threads * (bf16 ? 8 : 4);
  p.layers = (int)((vocab + per_layer - 1) / per_layer);
  auto kernel = halved ? sample_kernel<512, false> : sample_kernel<1024, false>;
  if (counted) kernel = halved ? sample_counts_kernel<512> : sample_counts_kernel<1024>;
  else if (bf16) kernel = halved ? sample_kernel<512, true> : sample_kernel<1024, true>;
  hipError_t e = hipSuccess;
  const int64_t most = host_most_groups(threads);
  for (int64_t r = 0; r < rows && e == hipSuccess; r += most) {
    p.logits = (const char*)logits + r * ld * (bf16 ? 2 : 4);
    p.u = u + r;
    p.tokens = tokens + r;
    p.probs = probs ? probs + r : nullptr;
    p.how = *how;
    if (how->temperature) p.how.temperature += r;
    if (how->top_k) p.how.top_k += r;
    if (how->top_p) p.how.top_p += r;
    if (how->min_p) p.how.min_p += r;
    kernel<<<(unsigned)(rows - r < most ? rows - r : most), threads, 0, (hipStream_t)stream>>>(p);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "sample launch: %s", hipGetErrorString(e));
}
