// mi_paged.hip -- attention of a chunk of new tokens over a paged K/V cache, gfx950.
//
// Row (token r, head h) of a sequence with n keys, at position p, reads the keys of KV head
// h / group:  O = sum_j e_j v_j / sum_j e_j,  e_j = exp(scale q.k_j - m),  j <= p (causal) or
// j < n, with the running maximum m and sum of an online softmax in fp32.
//
// One wave for each row: a lane scores one key of a 64-key step, then every lane sums two columns
// of V over the step's keys.
#include <hip/hip_runtime.h>
#include <math.h>

#include "mi_gemm_device.hpp"
#include "mi_paged.hpp"

namespace mig {
namespace {

struct AttnParams {
  PagedView pv;
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  const uint16_t *k, *v;
  int64_t q_t, q_h, o_t, o_h;
  int n_heads, group, d, causal, max_q;
  float scale;
};

__global__ void __launch_bounds__(64) paged_attn_row_kernel(AttnParams p) {
  __shared__ float qs[128], ps[64];
  const int lane = threadIdx.x;
  const int row = blockIdx.x / p.n_heads, h = blockIdx.x - row * p.n_heads, kvh = h / p.group;
  int s = row, q0 = row, n = 1;
  if (p.pv.q_start) {
    s = wave_first_false(p.pv.n_seqs, [&](int k) { return p.pv.q_start[k + 1] <= row; });
    if (s < p.pv.n_seqs) seq_rows(p.pv, s, q0, n);
  }
  if (s >= p.pv.n_seqs || row < q0 || row >= q0 + n || row - q0 >= p.max_q) return;
  const int64_t len = p.pv.kv_len[s], pos = len - n + (row - q0);
  int64_t end = p.causal ? pos + 1 : len;
  end = min(end, (int64_t)p.pv.max_pages << p.pv.page_shift);
  for (int c = lane; c < p.d; c += 64) qs[c] = bf16_bits_to_f32(p.q[row * p.q_t + h * p.q_h + c]);
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int64_t j0 = 0; j0 < end; j0 += 64) {
    const int64_t j = j0 + lane;
    const int page = j < end ? page_of(p.pv, s, j) : -1;
    const int64_t off = page * p.pv.page_stride + kvh * p.pv.head_stride +
                        (j & ((int64_t{1} << p.pv.page_shift) - 1)) * p.pv.slot_stride;
    float x = -INFINITY;
    if (page >= 0) {
      x = 0.0f;
      for (int c = 0; c < p.d; c += 8) {
        const u32x4_t w = *(const u32x4_t*)(p.k + off + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x += qs[c + 2 * e] * bf16_bits_to_f32(w[e]);
          x += qs[c + 2 * e + 1] * __uint_as_float(w[e] & 0xffff0000u);
        }
      }
      x *= p.scale;
    }
    float mx = x;
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) mx = fmaxf(mx, __shfl_xor(mx, i, 64));
    const float m_new = fmaxf(m, mx);
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float e = page >= 0 ? __expf(x - ref) : 0.0f, alpha = __expf(m - ref);
    float sum = e;
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) sum += __shfl_xor(sum, i, 64);
    m = m_new;
    l = l * alpha + sum;
    o0 *= alpha;
    o1 *= alpha;
    __syncthreads();
    ps[lane] = e;
    __syncthreads();
    const uint64_t there = __ballot(page >= 0);
    for (int i = 0; i < 64; ++i) {
      if (!(there >> i & 1)) continue;
      const int64_t at = __shfl(off, i, 64);
      if (2 * lane < p.d) {
        const uint32_t w = *(const uint32_t*)(p.v + at + 2 * lane);
        o0 += ps[i] * bf16_bits_to_f32(w);
        o1 += ps[i] * __uint_as_float(w & 0xffff0000u);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (2 * lane < p.d) *(uint32_t*)(p.o + row * p.o_t + h * p.o_h + 2 * lane) = pack_bf16x2(o0 * inv, o1 * inv);
  if (p.lse && lane == 0) p.lse[(int64_t)row * p.n_heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

size_t mi_paged_attn_workspace_size(int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t n_seqs, int64_t total_q,
                                    int64_t max_q_len, int64_t max_kv_len) {
  (void)n_heads, (void)n_kv, (void)head_dim, (void)n_seqs, (void)total_q, (void)max_q_len, (void)max_kv_len;
  return 0;
}

int mi_paged_attn(void* stream, const void* Q, int64_t q_t, int64_t q_h, void* O, int64_t o_t, int64_t o_h, float* lse,
                  int64_t n_heads, const mi_paged_cache* cache, const mi_paged_seqs* seqs, int64_t max_q_len,
                  int64_t max_kv_len, int32_t causal, float scale, void* workspace, size_t workspace_bytes) {
  int st = check_paged(cache, seqs);
  if (st != MI_OK) return st;
  if (n_heads < 0 || max_q_len < 0 || max_kv_len < 0) return host_fail(MI_ERR_SHAPE, "negative size");
  if (seqs->n_seqs == 0 || seqs->total_q == 0 || n_heads == 0 || max_q_len == 0) return MI_OK;
  if (cache->n_kv < 1 || n_heads % cache->n_kv || n_heads > 65536)
    return host_fail(MI_ERR_SHAPE, "n_heads=%lld is no multiple of n_kv=%lld", (long long)n_heads,
                     (long long)cache->n_kv);
  if (cache->head_dim > 128)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: at most 128", (long long)cache->head_dim);
  if (!Q || !O) return host_fail(MI_ERR_NULL, "Q or O is NULL");
  if (((uintptr_t)Q | (uintptr_t)O | (uintptr_t)workspace) & 15)
    return host_fail(MI_ERR_UNSUPPORTED, "Q, O and the workspace must be 16-byte aligned");
  if ((uintptr_t)lse & 3) return host_fail(MI_ERR_UNSUPPORTED, "lse must be aligned to its element size");
  if ((q_t | q_h | o_t | o_h) % 8) return host_fail(MI_ERR_UNSUPPORTED, "strides of Q and O must be multiples of 8");
  const int64_t d = cache->head_dim, rows = seqs->total_q;
  if ((rows > 1 && (o_t < d || q_t < 0)) || (n_heads > 1 && (o_h < d || q_h < 0)))
    return host_fail(MI_ERR_LD, "a stride of O is shorter than a row of %lld", (long long)d);
  if (Q == O && ((rows > 1 && q_t != o_t) || (n_heads > 1 && q_h != o_h)))
    return host_fail(MI_ERR_UNSUPPORTED, "in place needs the same strides of Q and O");
  if (!(scale > 0.0f) || !isfinite(scale)) return host_fail(MI_ERR_UNSUPPORTED, "scale must be positive and finite");
  if (rows * n_heads > INT32_MAX) return host_fail(MI_ERR_SHAPE, "total_q * n_heads exceeds 2^31-1");
  st = host_device();
  if (st != MI_OK) return st;
  (void)workspace_bytes;
  AttnParams p;
  p.pv = paged_view(cache, seqs);
  p.q = (const uint16_t*)Q;
  p.o = (uint16_t*)O;
  p.lse = lse;
  p.k = (const uint16_t*)cache->k;
  p.v = (const uint16_t*)cache->v;
  p.q_t = q_t, p.q_h = q_h, p.o_t = o_t, p.o_h = o_h;
  p.n_heads = (int)n_heads;
  p.group = (int)(n_heads / cache->n_kv);
  p.d = (int)d;
  p.causal = causal != 0;
  p.max_q = max_q_len > INT32_MAX ? INT32_MAX : (int)max_q_len;
  p.scale = scale;
  paged_attn_row_kernel<<<(unsigned)(rows * n_heads), 64, 0, (hipStream_t)stream>>>(p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "paged_attn launch: %s", hipGetErrorString(e));
}

}  // extern "C"
