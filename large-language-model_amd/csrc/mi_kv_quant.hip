// mi_kv_quant.hip -- new tokens into a paged K/V cache of 8 or 4 bits, and tokens read back from it, gfx950.
//
// A group is 32 neighbouring components of a head of a token.  With m = max |x|, its power of two is the least 2^e
// with m <= L 2^e, e >= -100, and a code is x / 2^e rounded to the nearest number of e4m3 (L = 464) or e2m1
// (L = 7).  L is half a step beyond the type's largest number (448, 6), so saturating the largest component
// costs no more than rounding it, and never does a group take twice the step for that.  e >= -100 keeps every
// value that the cache stands for, subnormal codes too, a normal bf16: reading back and attending round nothing.
//
// A code next to the border of two numbers would turn with the last bit of a rotation in 32 bits, so K is
// rotated in 64: the angle, its cosine and sine (once a token, for all heads), and the two products.  What is
// rounded to 32 bits on the way to the code is rounded to odd, so that the one rounding that counts is the last.
//
// Bound by HBM where there are many tokens, by the launch and a chain of tables, pages and rows where there are few.
// On an MI355X: 64 tokens appended in 4.0 us, 2100 of twelve prompts in 9.5 (23 MB; the rotation in 64 bits is 0.2 of
// them), 41000 read back in 21.2 (107 MB, 5.0 TB/s: a copy's rate).
#include <hip/hip_runtime.h>
#include <math.h>

#include "mi_kv_quant.hpp"
#include "mi_rope.hpp"

namespace mig {
namespace {

constexpr int KQ_THREADS = 256;
constexpr int KQ_MAX_TOKENS = 16;   // tokens of a workgroup of the append
constexpr int KQ_MAX_PAIRS = 1024;  // their cosines (and sines) in LDS, 16 KB
constexpr int KQ_MAX_DIM = 1024;    // head_dim: one token's pairs then always fit
constexpr int KR_MAX_TOKENS = 64;   // tokens of a workgroup of the reading back

// The cache as the kernels take it; strides of the codes are in the PagedView.
struct QuantView {
  uint8_t *k, *v, *ks, *vs;
  int64_t scale_page, scale_head, scale_slot;
};

// The first sequence from s on that ends behind token t (n_seqs: none), each lane on its own: steps of 1, 2, 4, .. until
// one does, and halves of the last step; the next sequence is one load away, any number of empty ones a few (two prompts of
// 2000 tokens side by side appended in 7.2 us, with 4000 empty sequences between them in 8.2; one by one 299).
__device__ __forceinline__ int first_after(const PagedView& pv, int s, int t) {
  int end = s;  // sequences before s end by t; `end` is looked at next
  for (int64_t step = 1; end < pv.n_seqs && pv.q_start[end + 1] <= t; step *= 2) {
    s = end + 1;
    end = (int)min((int64_t)s + step - 1, (int64_t)pv.n_seqs);
  }
  while (s < end) {  // in [s, end]
    const int mid = s + (end - s) / 2;
    if (pv.q_start[mid + 1] <= t) s = mid + 1;
    else end = mid;
  }
  return s;
}

// Tokens tok0 .. tok0 + n - 1 (n <= 64) looked up by the workgroup's first wave, one a lane: page (-1: none),
// slot and position in its sequence; page -2: a row of no sequence.
struct Tokens {
  int page[64], slot[64], pos[64];
};
__device__ __forceinline__ void look_up_tokens(const PagedView& pv, int64_t tok0, int n, Tokens& at) {
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x, t = (int)tok0 + min(lane, n - 1);
  int s = t, q0 = t, rows = 1;
  bool in = true;
  if (pv.q_start) {
    s = wave_first_false(pv.n_seqs, [&](int k) { return pv.q_start[k + 1] <= (int)tok0; });
    s = first_after(pv, s, t);
    in = s < pv.n_seqs;
    if (in) {
      seq_rows(pv, s, q0, rows);
      in = t >= q0 && t < q0 + rows;
    }
  }
  int64_t pos = 0;
  int page = -2;
  if (in) {
    pos = (int64_t)pv.kv_len[s] - rows + (t - q0);
    page = page_of(pv, s, pos);
  }
  if (lane < n) {
    at.page[lane] = page;
    at.slot[lane] = (int)(pos & ((int64_t{1} << pv.page_shift) - 1));
    at.pos[lane] = (int)pos;
  }
}

struct AppendParams {
  PagedView pv;
  QuantView c;
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  int64_t q_t, q_h, qo_t, qo_h, k_t, k_h, v_t, v_h;
  int n_heads, n_kv;  // 0: no Q, or no cache
  int d, rot, interleaved;
  float scale;
  const float* freq;  // null: nothing rotates
  const int32_t* pos;
  int tokens, per_wg;
  int64_t first;
};

// cos and sin of pos * f: n quarter turns and a rest of at most half of one to each side.  The product is rounded
// to 64 bits, its quotient by pi is not: 1/pi and the quotient are carried in two parts.
__device__ __forceinline__ void angle64(int64_t pos, float f, double& c, double& s) {
  constexpr double INV_PI = 0.31830988618379067154, INV_PI_LOW = -1.9678676675182486e-17;
  const double a = (double)pos * (double)f, turns = a * INV_PI;
  const double low = __builtin_fma(a, INV_PI, -turns) + a * INV_PI_LOW;
  const double n = rint(2.0 * turns);
  double sr, cr;
  sincospi(turns - 0.5 * n + low, &sr, &cr);
  const int q = (int)((int64_t)n & 3);
  c = (q & 1) ? sr : cr;
  s = (q & 1) ? cr : sr;
  if (q == 1 || q == 2) c = -c;
  if (q & 2) s = -s;
}

// x rounded to 32 bits toward odd: cut off, with the last bit set where something was.  Two bits wider than the
// codes at least, so rounding it to a code rounds x.
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  uint32_t u = __float_as_uint(f);
  const double back = (double)f;
  if (back == x || (u & 0x7f800000u) == 0x7f800000u) return f;
  if (fabs(back) > fabs(x)) --u;
  return __uint_as_float(u | 1u);
}

// Component c of x, rotated.
__device__ __forceinline__ float turned(const AppendParams& p, const uint16_t* x, int c, const double2* cs) {
  const float a = bf16_bits_to_f32(x[c]);
  if (c >= p.rot) return a;
  const int half = p.rot / 2;
  const bool second = p.interleaved ? c & 1 : c >= half;
  const int i = p.interleaved ? c >> 1 : second ? c - half : c;
  const float b = bf16_bits_to_f32(x[p.interleaved ? c ^ 1 : second ? c - half : c + half]);
  return to_odd((double)a * cs[i].x + (second ? (double)b : -(double)b) * cs[i].y);
}

// Four lanes side by side quantise a group, eight components y each, and write it: codes to `dst` (this lane's
// 4 or 8 bytes), the scale byte to `scale`.
template <int BITS>
__device__ __forceinline__ void write_group(const float (&y)[8], uint8_t* dst, uint8_t* scale) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);  // NaN above all
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
  // L = 1.75 * 2^2 or 1.8125 * 2^8
  constexpr uint32_t BELOW = BITS == 4 ? 2 : 8, TOP = BITS == 4 ? 0x600000 : 0x680000;
  const int from_m = (int)(m >> 23) - (int)BELOW + ((m & 0x7fffffu) > TOP ? 1 : 0);
  const bool none = m >= 0x7f000000u;
  const uint32_t byte = none ? 255u : (uint32_t)max(from_m, 27);
  [[maybe_unused]] const float inv = none ? 0.0f : __uint_as_float((254u - byte) << 23);
  uint32_t w[BITS / 4] = {};
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
#if defined(__HIP_DEVICE_COMPILE__)
    float a = none ? 0.0f : y[e] * inv, b = none ? 0.0f : y[e + 1] * inv;
    if constexpr (BITS == 4) {
      if (e == 0) w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], a, b, 1.0f, 0);
      if (e == 2) w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], a, b, 1.0f, 1);
      if (e == 4) w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], a, b, 1.0f, 2);
      if (e == 6) w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], a, b, 1.0f, 3);
    } else {
      a = fminf(fmaxf(a, -448.0f), 448.0f);  // beyond, the conversion gives NaN
      b = fminf(fmaxf(b, -448.0f), 448.0f);
      if (e & 2) w[e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)w[e / 4], true);
      else w[e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)w[e / 4], false);
    }
#endif
  }
  if constexpr (BITS == 4) *(uint32_t*)dst = w[0];
  else *(u32x2_t*)dst = u32x2_t{w[0], w[BITS / 4 - 1]};
  if ((threadIdx.x & 3) == 0) *scale = (uint8_t)byte;
}

// VEC: rows are whole 16-byte vectors and pairs lie in whole vectors.
template <int BITS, bool VEC>
__global__ void __launch_bounds__(KQ_THREADS) kv_append_quant_kernel(AppendParams p) {
  __shared__ double2 cs[KQ_MAX_PAIRS];
  __shared__ Tokens at;
  const int tid = threadIdx.x;
  const int64_t tok0 = p.first + (int64_t)blockIdx.x * p.per_wg;
  const int n_tok = (int)min((int64_t)p.per_wg, p.tokens - tok0);
  look_up_tokens(p.pv, tok0, n_tok, at);
  __syncthreads();
  const int half = p.rot / 2;
  for (int i = tid; i < n_tok * half; i += KQ_THREADS) {
    const int k = i / half;
    double c, s;
    angle64(p.pos ? p.pos[tok0 + k] : at.pos[k], p.freq[i - k * half], c, s);
    cs[i] = double2{c * p.scale, s * p.scale};
  }
  __syncthreads();

  // K and V: eight components a lane, the lanes of a group side by side
  const int runs = p.d / 8, kv_units = n_tok * 2 * p.n_kv * runs;
  // Q: a pair of vectors, as both turn together
  constexpr int W = VEC ? 8 : 1;
  const int q_runs = p.d / (2 * W), q_units = n_tok * p.n_heads * q_runs;
  for (int u = tid; u < kv_units + q_units; u += KQ_THREADS) {
    if (u < kv_units) {
      const int hh = u / runs, c0 = 8 * (u - hh * runs);
      const int k = hh / (2 * p.n_kv);
      int h = hh - k * 2 * p.n_kv;
      const bool is_v = h >= p.n_kv;
      if (is_v) h -= p.n_kv;
      const int page = at.page[k];
      if (page < 0) continue;
      const uint16_t* x = is_v ? p.v + (tok0 + k) * p.v_t + h * p.v_h : p.k + (tok0 + k) * p.k_t + h * p.k_h;
      const double2* pair = cs + k * half;
      float y[8];
      if constexpr (VEC) {
        RopeVec<uint16_t, 8> a;
        a.load(x + c0);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = a.v[e];
        if (!is_v && c0 < p.rot) {
          if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const double2 t = pair[(c0 + e) >> 1];
              y[e] = to_odd((double)a.v[e] * t.x + (e & 1 ? (double)a.v[e ^ 1] : -(double)a.v[e ^ 1]) * t.y);
            }
          } else {
            const bool second = c0 >= half;
            const int i = second ? c0 - half : c0;
            RopeVec<uint16_t, 8> b;
            b.load(x + (second ? i : c0 + half));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const double2 t = pair[i + e];
              y[e] = to_odd((double)a.v[e] * t.x + (second ? (double)b.v[e] : -(double)b.v[e]) * t.y);
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = is_v ? bf16_bits_to_f32(x[c0 + e]) : turned(p, x, c0 + e, pair);
      }
      const int slot = at.slot[k];
      uint8_t* dst = (is_v ? p.c.v : p.c.k) + page * p.pv.page_stride + h * p.pv.head_stride + slot * p.pv.slot_stride;
      uint8_t* sc = (is_v ? p.c.vs : p.c.ks) + page * p.c.scale_page + h * p.c.scale_head + slot * p.c.scale_slot;
      write_group<BITS>(y, dst + c0 * BITS / 8, sc + c0 / KV_GROUP);
      continue;
    }
    const int v = u - kv_units, hh = v / q_runs, ch = v - hh * q_runs;
    const int k = hh / p.n_heads, h = hh - k * p.n_heads;
    if (at.page[k] == -2) continue;
    const uint16_t* src = p.q + (tok0 + k) * p.q_t + h * p.q_h;
    uint16_t* dst = p.q_out + (tok0 + k) * p.qo_t + h * p.qo_h;
    const bool turn = ch < half / W;
    const int e0 = turn && !p.interleaved ? ch * W : ch * 2 * W;
    const int e1 = turn && !p.interleaved ? half + e0 : e0 + W;
    RopeVec<uint16_t, W> a, b;
    a.load(src + e0);
    b.load(src + e1);
    if (turn) {
      float c[W], s[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const double2 t = cs[k * half + ch * W + e];
        c[e] = (float)t.x, s[e] = (float)t.y;
      }
      rope_turn<W>(a.v, b.v, c, s, p.interleaved);
    }
    a.store(dst + e0);
    b.store(dst + e1);
  }
}

struct ReadParams {
  PagedView pv;
  QuantView c;
  void *k, *v;  // either may be null
  int64_t k_t, k_h, v_t, v_h;
  int n_kv, d, parts;  // parts: K and V, or one of them
  int tokens, per_wg;
  int64_t first;
};

// KR_COMPS components a lane, half a group: of half as many a lane's loads are 4 bytes (8 sequences of up
// to 16000 tokens in 4 bits: 27.4 us, so 21.0), of a group the stores of a wave lie 64 bytes apart (31.8).  T: uint16_t
// (bf16) or float; VEC: rows of the output are whole 16-byte vectors.
constexpr int KR_COMPS = 16;
template <int BITS, typename T, bool VEC>
__global__ void __launch_bounds__(KQ_THREADS) kv_read_quant_kernel(ReadParams p) {
  __shared__ Tokens at;
  const int64_t tok0 = p.first + (int64_t)blockIdx.x * p.per_wg;
  const int n_tok = (int)min((int64_t)p.per_wg, p.tokens - tok0);
  look_up_tokens(p.pv, tok0, n_tok, at);
  __syncthreads();
  const int runs = p.d / KR_COMPS, units = n_tok * p.parts * p.n_kv * runs;
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += KQ_THREADS) {
    const int hh = u / runs, c0 = KR_COMPS * (u - hh * runs);
    const int k = hh / (p.parts * p.n_kv);
    int h = hh - k * p.parts * p.n_kv;
    const bool is_v = h >= p.n_kv || !p.k;
    if (h >= p.n_kv) h -= p.n_kv;
    const int page = at.page[k], slot = at.slot[k];
    if (page == -2) continue;
    u32x4_t x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (page >= 0) {
      const uint8_t* src = (is_v ? p.c.v : p.c.k) + page * p.pv.page_stride + h * p.pv.head_stride +
                           slot * p.pv.slot_stride + c0 * BITS / 8;
      const uint8_t* sc = (is_v ? p.c.vs : p.c.ks) + page * p.c.scale_page + h * p.c.scale_head + slot * p.c.scale_slot;
      const float s = kv_power(sc[c0 / KV_GROUP]);
      uint32_t w[BITS / 2];
      if constexpr (BITS == 4) *(u32x2_t*)w = *(const u32x2_t*)src;
      else *(u32x4_t*)w = *(const u32x4_t*)src;
      x[0] = kv_eight<BITS>(w, s);
      x[1] = kv_eight<BITS>(w + BITS / 4, s);
    }
    T* dst = (T*)(is_v ? p.v : p.k) + (is_v ? (tok0 + k) * p.v_t + h * p.v_h : (tok0 + k) * p.k_t + h * p.k_h) + c0;
    if constexpr (sizeof(T) == 2 && VEC) {
      ((u32x4_t*)dst)[0] = x[0];
      ((u32x4_t*)dst)[1] = x[1];
    } else if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = x[i / 2][i % 2 * 2], b = x[i / 2][i % 2 * 2 + 1];
        ((f32x4_t*)dst)[i] = f32x4_t{__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u),
                                     __uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)};
      }
    } else {
#pragma unroll
      for (int e = 0; e < KR_COMPS; ++e) {
        const uint32_t w = x[e / 8][e % 8 / 2], bits = e & 1 ? w >> 16 : w & 0xffffu;
        if constexpr (sizeof(T) == 2) dst[e] = (T)bits;
        else dst[e] = __uint_as_float(bits << 16);
      }
    }
  }
}

QuantView quant_view(const mi_quant_cache* c) {
  return QuantView{(uint8_t*)c->k, (uint8_t*)c->v, (uint8_t*)c->k_scale, (uint8_t*)c->v_scale,
                   c->scale_page_stride, c->scale_head_stride, c->scale_slot_stride};
}

// Launches kernel(groups) for all of `tokens` in as many launches as their workgroups need.
template <class Params, class Launch>
int launch_tokens(Params& p, const char* what, Launch launch) {
  const int64_t groups = ((int64_t)p.tokens + p.per_wg - 1) / p.per_wg, most = host_most_groups(KQ_THREADS);
  for (int64_t g = 0; g < groups; g += most) {
    p.first = g * p.per_wg;
    launch((unsigned)(groups - g < most ? groups - g : most));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return host_fail(MI_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
  }
  return MI_OK;
}

// Tokens of a workgroup: about `each` units for a thread, but no fewer workgroups than two for each CU.
int tokens_of_group(int64_t tokens, int64_t units, int each, int most) {
  int64_t n = (int64_t)each * KQ_THREADS / (units > 0 ? units : 1);
  const int64_t spread = tokens / (2 * (int64_t)host_cus());
  if (n > spread) n = spread;
  return (int)(n < 1 ? 1 : n > most ? most : n);
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

int mi_kv_append_quant(void* stream, const void* q, int64_t q_t, int64_t q_h, void* q_out, int64_t qo_t, int64_t qo_h,
                       int64_t n_heads, const void* k, int64_t k_t, int64_t k_h, const void* v, int64_t v_t, int64_t v_h,
                       const mi_quant_cache* cache, const mi_paged_seqs* seqs, const mi_rotary* rotary) {
  int st = check_quant(cache, seqs);
  if (st != MI_OK) return st;
  if (n_heads < 0 || n_heads > 65536 || cache->n_kv > 65536)
    return host_fail(MI_ERR_SHAPE, "n_heads=%lld, n_kv=%lld", (long long)n_heads, (long long)cache->n_kv);
  if (rotary && (st = check_rotary(rotary, cache->head_dim)) != MI_OK) return st;
  if (seqs->total_q == 0 || seqs->n_seqs == 0) return MI_OK;
  if (cache->head_dim > KQ_MAX_DIM)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: at most %d", (long long)cache->head_dim, KQ_MAX_DIM);
  if (q && !q_out) return host_fail(MI_ERR_NULL, "q_out is NULL");
  if (cache->n_kv > 0 && (!k || !v)) return host_fail(MI_ERR_NULL, "k or v is NULL");
  if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) % 2)
    return host_fail(MI_ERR_UNSUPPORTED, "pointers must be aligned to their element size");
  const int64_t tokens = seqs->total_q;
  if (q && ((tokens > 1 && qo_t == 0) || (n_heads > 1 && qo_h == 0)))
    return host_fail(MI_ERR_LD, "a stride of q_out is 0: rows would share memory");
  if (q && q == q_out && ((tokens > 1 && q_t != qo_t) || (n_heads > 1 && q_h != qo_h)))
    return host_fail(MI_ERR_UNSUPPORTED, "in place needs the same strides of q and q_out");
  AppendParams p = {};
  p.pv = paged_view(cache, seqs);
  p.c = quant_view(cache);
  p.n_heads = q ? (int)n_heads : 0;
  p.n_kv = cache->num_pages > 0 ? (int)cache->n_kv : 0;
  if (p.n_heads + p.n_kv == 0) return MI_OK;
  st = host_device();
  if (st != MI_OK) return st;
  p.q = (const uint16_t*)q, p.k = (const uint16_t*)k, p.v = (const uint16_t*)v;
  p.q_out = (uint16_t*)q_out;
  p.q_t = q_t, p.q_h = q_h, p.qo_t = qo_t, p.qo_h = qo_h;
  p.k_t = k_t, p.k_h = k_h, p.v_t = v_t, p.v_h = v_h;
  p.d = (int)cache->head_dim;
  p.rot = rotary ? (int)rotary->rot_dim : 0;
  p.interleaved = rotary ? rotary->interleaved : 0;
  p.scale = rotary ? rotary->scale : 1.0f;
  p.freq = rotary ? rotary->inv_freq : nullptr;
  p.pos = rotary ? rotary->positions : nullptr;
  p.tokens = (int)tokens;
  // pairs of vectors: 16 components, and every row on a 16-byte boundary
  bool vec = p.rot % 16 == 0;
  auto rows_fit = [&](const void* at, int64_t t, int64_t h, int64_t heads) {
    return (uintptr_t)at % 16 == 0 && (tokens <= 1 || t % 8 == 0) && (heads <= 1 || h % 8 == 0);
  };
  if (p.n_heads) vec = vec && rows_fit(q, q_t, q_h, n_heads) && rows_fit(q_out, qo_t, qo_h, n_heads);
  if (p.n_kv) vec = vec && rows_fit(k, k_t, k_h, p.n_kv) && rows_fit(v, v_t, v_h, p.n_kv);
  const int64_t units = (int64_t)p.n_kv * 2 * (p.d / 8) + (int64_t)p.n_heads * (p.d / (vec ? 16 : 2));
  p.per_wg = tokens_of_group(tokens, units, 3, KQ_MAX_TOKENS);
  if (p.rot) p.per_wg = p.per_wg < KQ_MAX_PAIRS / (p.rot / 2) ? p.per_wg : KQ_MAX_PAIRS / (p.rot / 2);
  hipStream_t hs = (hipStream_t)stream;
  const bool four = cache->format == MI_KV_E2M1;
  return launch_tokens(p, "kv_append_quant", [&](unsigned grid) {
    if (four && vec) kv_append_quant_kernel<4, true><<<grid, KQ_THREADS, 0, hs>>>(p);
    else if (four) kv_append_quant_kernel<4, false><<<grid, KQ_THREADS, 0, hs>>>(p);
    else if (vec) kv_append_quant_kernel<8, true><<<grid, KQ_THREADS, 0, hs>>>(p);
    else kv_append_quant_kernel<8, false><<<grid, KQ_THREADS, 0, hs>>>(p);
  });
}

int mi_kv_read_quant(void* stream, void* k, int64_t k_t, int64_t k_h, void* v, int64_t v_t, int64_t v_h, int32_t dtype,
                     const mi_quant_cache* cache, const mi_paged_seqs* seqs) {
  int st = check_quant(cache, seqs);
  if (st != MI_OK) return st;
  if (dtype != MI_BF16 && dtype != MI_F32) return host_fail(MI_ERR_DTYPE, "dtype %d", dtype);
  if (cache->n_kv > 65536) return host_fail(MI_ERR_SHAPE, "n_kv=%lld", (long long)cache->n_kv);
  if (seqs->total_q == 0 || seqs->n_seqs == 0 || cache->n_kv == 0 || (!k && !v)) return MI_OK;
  if (cache->head_dim > KQ_MAX_DIM)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: at most %d", (long long)cache->head_dim, KQ_MAX_DIM);
  const int64_t tokens = seqs->total_q, es = dtype == MI_BF16 ? 2 : 4, d = cache->head_dim;
  if (((uintptr_t)k | (uintptr_t)v) % (uintptr_t)es)
    return host_fail(MI_ERR_UNSUPPORTED, "pointers must be aligned to their element size");
  for (int i = 0; i < 2; ++i) {
    if (!(i ? v : k)) continue;
    if ((tokens > 1 && (i ? v_t : k_t) < d) || (cache->n_kv > 1 && (i ? v_h : k_h) < d))
      return host_fail(MI_ERR_LD, "a stride of %s is shorter than a row of %lld", i ? "v" : "k", (long long)d);
  }
  st = host_device();
  if (st != MI_OK) return st;
  ReadParams p = {};
  p.pv = paged_view(cache, seqs);
  p.c = quant_view(cache);
  p.k = k, p.v = v;
  p.k_t = k_t, p.k_h = k_h, p.v_t = v_t, p.v_h = v_h;
  p.n_kv = (int)cache->n_kv;
  p.d = (int)d;
  p.parts = k && v ? 2 : 1;
  p.tokens = (int)tokens;
  auto rows_fit = [&](const void* at, int64_t t, int64_t h) {
    return !at || ((uintptr_t)at % 16 == 0 && (tokens <= 1 || t * es % 16 == 0) && (p.n_kv <= 1 || h * es % 16 == 0));
  };
  const bool vec = rows_fit(k, k_t, k_h) && rows_fit(v, v_t, v_h), four = cache->format == MI_KV_E2M1;
  p.per_wg = tokens_of_group(tokens, (int64_t)p.parts * p.n_kv * (d / KR_COMPS), 4, KR_MAX_TOKENS);
  hipStream_t hs = (hipStream_t)stream;
  return launch_tokens(p, "kv_read_quant", [&](unsigned grid) {
    if (dtype == MI_BF16) {
      if (four && vec) kv_read_quant_kernel<4, uint16_t, true><<<grid, KQ_THREADS, 0, hs>>>(p);
      else if (four) kv_read_quant_kernel<4, uint16_t, false><<<grid, KQ_THREADS, 0, hs>>>(p);
      else if (vec) kv_read_quant_kernel<8, uint16_t, true><<<grid, KQ_THREADS, 0, hs>>>(p);
      else kv_read_quant_kernel<8, uint16_t, false><<<grid, KQ_THREADS, 0, hs>>>(p);
    } else {
      if (four && vec) kv_read_quant_kernel<4, float, true><<<grid, KQ_THREADS, 0, hs>>>(p);
      else if (four) kv_read_quant_kernel<4, float, false><<<grid, KQ_THREADS, 0, hs>>>(p);
      else if (vec) kv_read_quant_kernel<8, float, true><<<grid, KQ_THREADS, 0, hs>>>(p);
      else kv_read_quant_kernel<8, float, false><<<grid, KQ_THREADS, 0, hs>>>(p);
    }
  });
}

}  // extern "C"
