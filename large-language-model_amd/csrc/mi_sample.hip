// mi_sample.hip -- one token for each row of logits, by temperature, top-k, top-p and min-p, gfx950.
//
// With the tokens of a row ordered by (logit descending, index ascending), each of the three
// filters keeps a run from the front, so what is kept is fixed by one border: a logit and how many
// of the tokens equal to it.  A row needs no sort: the border is found digit by digit in the
// logits' bits (an order-preserving integer key), by counting tokens above (top-k) or summing their
// weights (top-p).
//
// Weights w = exp((x - max) / T) are computed in 64 bits and held as integers, w * 2^shift, so every
// sum is exact: it is the same whatever order atomics and waves add in, and a border is never moved
// by rounding.  A weight below half of 2^-shift counts as nothing: u = 0, one of 2^24 numbers, then does
// not draw a token whose chance is 1e-20.
//
// One workgroup a row.
#include <hip/hip_runtime.h>
#include <math.h>

#include "mi_gemm_device.hpp"
#include "mi_host.hpp"

namespace mig {
namespace {

constexpr int SMP_THREADS = 1024;
constexpr int SMP_WAVES = SMP_THREADS / 64;
constexpr uint32_t SMP_KEY_NEG_INF = 0x007fffffu;  // key of -inf: nothing below it is a token

struct SampleParams {
  const void* logits;
  int64_t ld;
  int vocab, shift;
  const float* u;
  int32_t* tokens;
  float* probs;
  mi_sampling how;
};

// Keys order as the logits do; both zeros have one key, NaN the lowest.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0;
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

template <bool BF16>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  if constexpr (BF16) return bf16_bits_to_f32(((const uint16_t*)row)[i]);
  else return ((const float*)row)[i];
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct RowWeights {
  float mx;
  double inv_t, one;  // 1 / T, 2^shift
  __device__ __forceinline__ uint64_t of(float x) const {
    if (x == mx) return (uint64_t)one;
    if (!(x > -INFINITY) || mx == INFINITY) return 0;
    return (uint64_t)rint(exp(((double)x - (double)mx) * inv_t) * one);
  }
};

template <bool BF16>
__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(SampleParams p) {
  __shared__ uint32_t cnt[256];
  __shared__ uint64_t mass[256];
  __shared__ uint64_t wave_mass[SMP_WAVES];
  __shared__ uint32_t wave_cnt[SMP_WAVES];
  __shared__ uint32_t s_key, s_left;
  __shared__ uint64_t s_mass;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int V = p.vocab;
  const void* x = (const char*)p.logits + (int64_t)row * p.ld * (BF16 ? 2 : 4);

  float T = p.how.temperature ? p.how.temperature[row] : p.how.temperature_all;
  int top_k = p.how.top_k ? p.how.top_k[row] : p.how.top_k_all;
  const float top_p = p.how.top_p ? p.how.top_p[row] : p.how.top_p_all;
  const float min_p = p.how.min_p ? p.how.min_p[row] : p.how.min_p_all;
  if (!(T > 0.0f)) {
    T = 1.0f;
    top_k = 1;
  }

  uint32_t mk = 0;
  for (int i = tid; i < V; i += SMP_THREADS) mk = max(mk, key_of(logit_at<BF16>(x, i)));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
  if (lane == 0) wave_cnt[wave] = mk;
  __syncthreads();
  for (int w = 0; w < SMP_WAVES; ++w) mk = max(mk, wave_cnt[w]);
  if (mk <= SMP_KEY_NEG_INF) {
    if (tid == 0) {
      p.tokens[row] = -1;
      if (p.probs) p.probs[row] = 0.0f;
    }
    return;
  }
  const RowWeights W = {logit_of(mk), 1.0 / (double)T, (double)(uint64_t{1} << p.shift)};

  // Kept so far: keys above `border`, and the first `ties` tokens that equal it.
  uint32_t border = SMP_KEY_NEG_INF, ties = 0;

  // Narrows the kept run to its first tokens, `want` of them (by_mass false), or as many as
  // reach the weight `goal`.
  auto narrow = [&](bool by_mass, uint32_t want, uint64_t goal) {
    uint32_t prefix = 0, above = 0;  // digits found; tokens above them
    uint64_t above_m = 0;
    for (int sh = 24; sh >= 0; sh -= 8) {
      __syncthreads();
      if (tid < 256) cnt[tid] = 0, mass[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += SMP_THREADS) {
        const float xi = logit_at<BF16>(x, i);
        const uint32_t k = key_of(xi);
        if (k <= border || (sh < 24 && (k ^ prefix) >> (sh + 8))) continue;
        const int b = k >> sh & 255;
        atomicAdd(&cnt[b], 1u);
        if (by_mass) atomicAdd((unsigned long long*)&mass[b], (unsigned long long)W.of(xi));
      }
      __syncthreads();
      if (tid == 0) {
        // tokens that equal the old border stand in its bin, kept ones only
        if (ties && (sh == 24 || !((border ^ prefix) >> (sh + 8)))) {
          cnt[border >> sh & 255] += ties;
          mass[border >> sh & 255] += ties * W.of(logit_of(border));
        }
        uint32_t c = above;
        uint64_t m = above_m;
        int b = 255;
        for (; b > 0; --b) {
          if (by_mass ? m + mass[b] >= goal : c + cnt[b] >= want) break;
          c += cnt[b];
          m += mass[b];
        }
        s_key = prefix | (uint32_t)b << sh;
        s_left = c;
        s_mass = m;
      }
      __syncthreads();
      prefix = s_key;
      above = s_left;
      above_m = s_mass;
    }
    // all tokens above `prefix` are kept, and some that equal it
    if (by_mass) {
      const uint64_t w = W.of(logit_of(prefix));
      uint64_t n = w ? (goal > above_m ? (goal - above_m + w - 1) / w : 0) : 0;
      if (n > (uint64_t)V) n = V;
      const uint32_t most = prefix == border ? ties : 0xffffffffu;
      border = prefix;
      ties = n < most ? (uint32_t)n : most;
    } else {
      const uint32_t n = want - above, most = prefix == border ? ties : 0xffffffffu;
      border = prefix;
      ties = n < most ? n : most;
    }
  };

  // Weight of what is kept: this wave's share of the row, a run of whole 64s, in index order.
  const int run = (V + SMP_WAVES * 64 - 1) / (SMP_WAVES * 64) * 64;
  const int i0 = min(wave * run, V), i1 = min(i0 + run, V);
  uint32_t floor_key = 0;  // min_p: keys below it are dropped
  uint64_t total = 0, before = 0;
  uint32_t ties_before = 0;
  auto sum_kept = [&]() {
    uint64_t m = 0;
    uint32_t c = 0;
    for (int i = i0 + lane; i < i1; i += 64) {
      const float xi = logit_at<BF16>(x, i);
      const uint32_t k = key_of(xi);
      if (k > border && k >= floor_key) m += W.of(xi);
      c += k == border;
    }
    m = wave_sum_u64(m);
    c = (uint32_t)wave_sum_u64(c);
    __syncthreads();
    if (lane == 0) wave_mass[wave] = m, wave_cnt[wave] = c;
    __syncthreads();
    const uint64_t wb = border >= floor_key ? W.of(logit_of(border)) : 0;
    uint32_t seen = 0;
    total = 0;
    for (int w = 0; w < SMP_WAVES; ++w) {
      if (w == wave) before = total, ties_before = seen;
      const uint32_t left = ties > seen ? ties - seen : 0;
      total += wave_mass[w] + wb * min(left, wave_cnt[w]);
      seen += wave_cnt[w];
    }
  };

  if (top_k > 0 && top_k < V) narrow(false, (uint32_t)top_k, 0);
  if (top_p < 1.0f) {
    sum_kept();
    const double goal = ceil((double)top_p * (double)total);
    narrow(true, 0, goal >= 1.0 ? (uint64_t)goal : 1);
  }
  if (min_p > 0.0f) {
    // the lowest key whose weight reaches min_p; the largest logit always stays
    const double low = (double)min_p * W.one;
    uint32_t lo = SMP_KEY_NEG_INF, hi = mk;  // below(lo), not below(hi)
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const float xm = logit_of(mid);
      const double w = xm == W.mx ? W.one : exp(((double)xm - (double)W.mx) * W.inv_t) * W.one;
      if (w >= low) hi = mid;
      else lo = mid;
    }
    floor_key = hi;
  }
  sum_kept();

  // the token at which the kept weight passes u * total
  const double t = (double)p.u[row] * (double)total;
  uint64_t target = t > 0.0 ? (uint64_t)t : 0;
  if (target >= total) target = total - 1;
  const uint64_t wb = border >= floor_key ? W.of(logit_of(border)) : 0;
  uint64_t acc = before;
  uint32_t seen = ties_before;
  for (int j0 = i0; j0 < i1; j0 += 64) {
    const int i = j0 + lane;
    const float xi = i < i1 ? logit_at<BF16>(x, i) : -INFINITY;
    const uint32_t k = i < i1 ? key_of(xi) : 0;
    const bool tie = i < i1 && k == border;
    const uint64_t tb = __ballot(tie);
    const uint32_t rank = seen + (uint32_t)__popcll(tb & ((uint64_t{1} << lane) - 1));
    uint64_t w = k > border && k >= floor_key ? W.of(xi) : tie && rank < ties ? wb : 0;
    const uint64_t own_w = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = __shfl_up(w, o, 64);
      if (lane >= o) w += y;
    }
    const uint64_t hit = __ballot(acc + w > target && acc + w - own_w <= target);
    if (hit) {
      if (lane == (int)__ffsll((unsigned long long)hit) - 1) {
        p.tokens[row] = i;
        if (p.probs) p.probs[row] = (float)((double)own_w / (double)total);
      }
      break;
    }
    acc += __shfl(w, 63, 64);
    seen += (uint32_t)__popcll(tb);
  }
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
  p.shift = 62 - bits < 52 ? 62 - bits : 52;
  p.u = u;
  p.tokens = tokens;
  p.probs = probs;
  p.how = *how;
  if (dtype == MI_BF16) sample_kernel<true><<<(unsigned)rows, SMP_THREADS, 0, (hipStream_t)stream>>>(p);
  else sample_kernel<false><<<(unsigned)rows, SMP_THREADS, 0, (hipStream_t)stream>>>(p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "sample launch: %s", hipGetErrorString(e));
}
