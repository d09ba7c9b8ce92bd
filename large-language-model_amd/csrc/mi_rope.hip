// mi_rope.hip -- rotary positions and the append to a paged cache, gfx950.
//
// Pair i of a head at position p turns by the angle p * inv_freq[i]:
//   a' = scale (a cos - b sin),  b' = scale (b cos + a sin)
// with (a, b) = (x[i], x[i + rot/2]) or (x[2i], x[2i+1]); the way back is the transposed map, the
// same with the sine negated.  Three operations for each element that is read and written once:
// bound by HBM.  8 x 1024 tokens of 16 + 2 x 4 heads of 128, bf16, there and back: 201 MB in 37 us
// from the caches behind L2, 43 from memory, where a copy of 1 GiB takes 40 for as much; 16381 tokens
// with interleaved pairs 33 and 41.  A decode step's append (64 tokens) takes 4 us, its launch.
//
// A workgroup takes a few tokens with all heads of all tensors.  It first computes each token's
// cosines and sines once into LDS, where every head of the token reads them: 64 pairs of a
// 128-component head cost 64 sine and cosine pairs a token instead of 64 for each head.  The angle
// is a product in 64 bits, brought into [-1/2, 1/2] half turns before it is rounded to 32: a
// 32-bit product at position 10^6 is off by 0.06 rad, this by 1e-7 at any position.
// Then each thread moves units of VEC pairs: two vectors of VEC elements, which a half layout finds
// rot/2 apart and an interleaved one side by side.  Only the thread that read a unit writes it,
// after all its reads, so a tensor may be rotated in place.
#include <hip/hip_runtime.h>
#include <math.h>

#include "mi_rope.hpp"

namespace mig {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_TOKENS = 16;   // tokens of a workgroup
constexpr int ROPE_MAX_PAIRS = 1024;  // cosines (and sines) of a workgroup in LDS, 8 KB
constexpr int ROPE_MAX_DIM = 1024;    // head_dim: one token's pairs then always fit

struct RopePart {
  const void* src;
  void* dst;
  int64_t sb, st, sh, db, dt, dh;  // elements
  int first;                       // its first head among all heads of the call
  int rotate;
  int paged;                       // dst is the cache: the token's offset stands in for db and dt
};

struct RopeParams {
  RopePart part[4];
  int n_parts, heads;   // heads of all parts together
  int d, rot, interleaved;
  float scale, sign;
  const float* freq;    // null: nothing rotates
  const int32_t* pos;
  int64_t pos_ld, pos0;
  int tokens, T;        // T: tokens of a sequence (dense)
  int per_wg;           // tokens of a workgroup
  int64_t first;        // the launch's first token
  PagedView pv;
};

// cos and sin of pos * f: n quarter turns and a rest of at most a quarter turn to each side.
__device__ __forceinline__ void rope_angle(int64_t pos, float f, float& c, float& s) {
  const double half_turns = (double)pos * (double)f * 0.31830988618379067154;
  const double n = rint(2.0 * half_turns);
  const float r = (float)(half_turns - 0.5 * n);
  float sr, cr;
  sincospif(r, &sr, &cr);
  const int q = (int)((int64_t)n & 3);
  c = (q & 1) ? sr : cr;
  s = (q & 1) ? cr : sr;
  if (q == 1 || q == 2) c = -c;
  if (q & 2) s = -s;
}

// T: float, or uint16_t holding bf16 bits.
template <typename T, int VEC, bool PAGED>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(RopeParams p) {
  __shared__ float cs[ROPE_MAX_PAIRS], sn[ROPE_MAX_PAIRS];
  __shared__ int64_t tok_pos[ROPE_MAX_TOKENS], tok_off[ROPE_MAX_TOKENS];
  __shared__ int tok_b[ROPE_MAX_TOKENS], tok_t[ROPE_MAX_TOKENS];
  const int tid = threadIdx.x;
  const int64_t tok0 = p.first + (int64_t)blockIdx.x * p.per_wg;
  const int n_tok = (int)min((int64_t)p.per_wg, p.tokens - tok0);

  if constexpr (PAGED) {
    for (int i = tid >> 6; i < n_tok; i += ROPE_THREADS / 64) {
      const int t = (int)tok0 + i;
      int s = t, q0 = t, n = 1;
      if (p.pv.q_start) {
        s = wave_first_false(p.pv.n_seqs, [&](int k) { return p.pv.q_start[k + 1] <= t; });
        if (s < p.pv.n_seqs) seq_rows(p.pv, s, q0, n);
      }
      if ((tid & 63) == 0) {
        int64_t pos = 0, off = -1;
        const bool in = s < p.pv.n_seqs && t >= q0 && t < q0 + n;
        if (in) {
          pos = (int64_t)p.pv.kv_len[s] - n + (t - q0);
          const int page = page_of(p.pv, s, pos);
          if (page >= 0)
            off = page * p.pv.page_stride + (pos & ((int64_t{1} << p.pv.page_shift) - 1)) * p.pv.slot_stride;
          if (p.pos) pos = p.pos[t];
        }
        tok_pos[i] = pos;
        tok_off[i] = off;
        tok_b[i] = in ? 0 : -1;
        tok_t[i] = t;
      }
    }
  } else if (tid < n_tok) {
    const int g = (int)tok0 + tid, b = g / p.T, t = g - b * p.T;
    tok_b[tid] = b;
    tok_t[tid] = t;
    tok_pos[tid] = p.pos ? (int64_t)p.pos[b * p.pos_ld + t] : p.pos0 + t;
  }
  __syncthreads();
  const int half = p.rot / 2;
  for (int i = tid; i < n_tok * half; i += ROPE_THREADS) {
    const int k = i / half;
    float c, s;
    rope_angle(tok_pos[k], p.freq[i - k * half], c, s);
    cs[i] = c * p.scale;
    sn[i] = s * p.scale * p.sign;
  }
  __syncthreads();

  const int per_head = p.d / (2 * VEC), turning = half / VEC;
  const int units = n_tok * p.heads * per_head;
  for (int u = tid; u < units; u += ROPE_THREADS) {
    const int hh = u / per_head, ch = u - hh * per_head;
    const int k = hh / p.heads;
    int h = hh - k * p.heads, which = 0;
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (i < p.n_parts && h >= p.part[i].first) which = i;
    const RopePart& r = p.part[which];
    h -= r.first;
    if (PAGED && (tok_b[k] < 0 || (r.paged && tok_off[k] < 0))) continue;
    const T* src = (const T*)r.src + tok_b[k] * r.sb + tok_t[k] * r.st + h * r.sh;
    T* dst = (T*)r.dst + h * r.dh;
    if (PAGED && r.paged) dst += tok_off[k];
    else dst += tok_b[k] * r.db + tok_t[k] * r.dt;
    const bool turn = r.rotate && ch < turning;
    const int e0 = turn && !p.interleaved ? ch * VEC : ch * 2 * VEC;
    const int e1 = turn && !p.interleaved ? half + e0 : e0 + VEC;
    RopeVec<T, VEC> a, b;
    a.load(src + e0);
    b.load(src + e1);
    if (turn) {
      const float* c = cs + k * half + ch * VEC;
      const float* s = sn + k * half + ch * VEC;
      rope_turn<VEC>(a.v, b.v, c, s, p.interleaved);
    }
    a.store(dst + e0);
    b.store(dst + e1);
  }
}

// Can units of `vec` pairs move every part?
bool rope_vec_fits(const RopeParams& p, int vec, int es, int64_t batch, int64_t seq_len, const int* heads) {
  if (p.d % (2 * vec) || p.rot % (2 * vec)) return false;
  for (int i = 0; i < p.n_parts; ++i) {
    const RopePart& r = p.part[i];
    if (heads[i] == 0) continue;
    if (((uintptr_t)r.src | (uintptr_t)r.dst) % (uintptr_t)(vec * es)) return false;
    if (batch > 1 && (r.sb % vec || r.db % vec)) return false;
    if (seq_len > 1 && (r.st % vec || r.dt % vec)) return false;
    if (heads[i] > 1 && (r.sh % vec || r.dh % vec)) return false;
  }
  return true;
}

template <typename T, int VEC>
hipError_t rope_launch(RopeParams p, bool paged, hipStream_t st) {
  const int64_t groups = ((int64_t)p.tokens + p.per_wg - 1) / p.per_wg, most = host_most_groups(ROPE_THREADS);
  hipError_t e = hipSuccess;
  for (int64_t g = 0; g < groups && e == hipSuccess; g += most) {
    const unsigned grid = (unsigned)(groups - g < most ? groups - g : most);
    p.first = g * p.per_wg;
    if (paged) rope_kernel<T, VEC, true><<<grid, ROPE_THREADS, 0, st>>>(p);
    else rope_kernel<T, VEC, false><<<grid, ROPE_THREADS, 0, st>>>(p);
    e = hipGetLastError();
  }
  return e;
}

// Fills in the workgroup's share and launches; heads: of each part.
int rope_run(RopeParams& p, bool paged, bool bf16, int64_t batch, int64_t seq_len, const int* heads, void* stream) {
  int st = host_device();
  if (st != MI_OK) return st;
  const int es = bf16 ? 2 : 4;
  int vec = bf16 ? 8 : 4;
  while (vec > 1 && !rope_vec_fits(p, vec, es, batch, seq_len, heads)) vec = vec == 8 ? 4 : 1;
  // three units of each thread, but no fewer workgroups than two for each CU
  const int64_t units = (int64_t)p.heads * (p.d / (2 * vec));
  int64_t n = 3 * ROPE_THREADS / (units > 0 ? units : 1);
  const int64_t spread = p.tokens / (2 * (int64_t)host_cus());
  if (n > spread) n = spread;
  if (p.rot && n > ROPE_MAX_PAIRS / (p.rot / 2)) n = ROPE_MAX_PAIRS / (p.rot / 2);
  p.per_wg = (int)(n < 1 ? 1 : n > ROPE_MAX_TOKENS ? ROPE_MAX_TOKENS : n);
  hipError_t e;
  hipStream_t hs = (hipStream_t)stream;
  if (bf16)
    e = vec == 8 ? rope_launch<uint16_t, 8>(p, paged, hs)
                 : vec == 4 ? rope_launch<uint16_t, 4>(p, paged, hs) : rope_launch<uint16_t, 1>(p, paged, hs);
  else
    e = vec == 4 ? rope_launch<float, 4>(p, paged, hs) : rope_launch<float, 1>(p, paged, hs);
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "rope launch: %s", hipGetErrorString(e));
}

void set_rotary(RopeParams& p, const mi_rotary* r, bool inverse) {
  p.rot = r ? (int)r->rot_dim : 0;
  p.interleaved = r ? r->interleaved : 0;
  p.scale = r ? r->scale : 1.0f;
  p.sign = inverse ? -1.0f : 1.0f;
  p.freq = r ? r->inv_freq : nullptr;
  p.pos = r ? r->positions : nullptr;
  p.pos_ld = r ? r->positions_ld : 0;
  p.pos0 = r ? r->pos0 : 0;
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

int mi_rope(void* stream, const mi_rope_part* parts, int64_t n_parts, int64_t batch, int64_t seq_len,
            int64_t head_dim, const mi_rotary* rotary, int32_t inverse, int32_t dtype) {
  if (batch < 0 || seq_len < 0 || head_dim < 0) return host_fail(MI_ERR_SHAPE, "negative size");
  if (n_parts < 1 || n_parts > 4) return host_fail(MI_ERR_SHAPE, "n_parts=%lld: 1 to 4 are possible", (long long)n_parts);
  if (!parts || !rotary) return host_fail(MI_ERR_NULL, "parts or rotary is NULL");
  if (dtype != MI_F32 && dtype != MI_BF16) return host_fail(MI_ERR_DTYPE, "dtype %d", dtype);
  if (batch > INT32_MAX || seq_len > INT32_MAX || (batch && seq_len > INT32_MAX / batch))
    return host_fail(MI_ERR_SHAPE, "batch * seq_len exceeds 2^31-1");
  if (head_dim % 2 || head_dim > ROPE_MAX_DIM)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: an even number up to %d is needed", (long long)head_dim,
                     ROPE_MAX_DIM);
  int64_t heads = 0;
  for (int64_t i = 0; i < n_parts; ++i) {
    if (parts[i].heads < 0 || parts[i].heads > 65536)
      return host_fail(MI_ERR_SHAPE, "part %lld: heads=%lld", (long long)i, (long long)parts[i].heads);
    heads += parts[i].heads;
  }
  if (batch == 0 || seq_len == 0 || head_dim == 0 || heads == 0) return MI_OK;
  int st = check_rotary(rotary, head_dim);
  if (st != MI_OK) return st;
  RopeParams p = {};
  int n_heads[4] = {};
  const uintptr_t es = dtype == MI_BF16 ? 2 : 4;
  for (int64_t i = 0; i < n_parts; ++i) {
    const mi_rope_part& a = parts[i];
    RopePart& r = p.part[i];
    if (a.reserved != 0) return host_fail(MI_ERR_SHAPE, "part %lld: reserved must be 0", (long long)i);
    n_heads[i] = (int)a.heads;
    r.first = p.heads;
    p.heads += (int)a.heads;
    if (a.heads == 0) continue;
    if (!a.src || !a.dst) return host_fail(MI_ERR_NULL, "part %lld: src or dst is NULL", (long long)i);
    if (((uintptr_t)a.src | (uintptr_t)a.dst) % es)
      return host_fail(MI_ERR_UNSUPPORTED, "part %lld: pointers must be aligned to their element size", (long long)i);
    if ((batch > 1 && a.dst_b == 0) || (seq_len > 1 && a.dst_t == 0) || (a.heads > 1 && a.dst_h == 0))
      return host_fail(MI_ERR_LD, "part %lld: a stride of dst is 0: rows would share memory", (long long)i);
    if (a.src == a.dst && ((batch > 1 && a.src_b != a.dst_b) || (seq_len > 1 && a.src_t != a.dst_t) ||
                           (a.heads > 1 && a.src_h != a.dst_h)))
      return host_fail(MI_ERR_UNSUPPORTED, "part %lld: in place needs the same strides", (long long)i);
    r.src = a.src;
    r.dst = a.dst;
    r.sb = a.src_b, r.st = a.src_t, r.sh = a.src_h;
    r.db = a.dst_b, r.dt = a.dst_t, r.dh = a.dst_h;
    r.rotate = a.rotate != 0;
  }
  p.n_parts = (int)n_parts;
  p.d = (int)head_dim;
  p.tokens = (int)(batch * seq_len);
  p.T = (int)seq_len;
  set_rotary(p, rotary, inverse != 0);
  return rope_run(p, false, dtype == MI_BF16, batch, seq_len, n_heads, stream);
}

int mi_kv_append(void* stream, const void* q, int64_t q_t, int64_t q_h, void* q_out, int64_t qo_t, int64_t qo_h,
                 int64_t n_heads, const void* k, int64_t k_t, int64_t k_h, const void* v, int64_t v_t, int64_t v_h,
                 const mi_paged_cache* cache, const mi_paged_seqs* seqs, const mi_rotary* rotary) {
  int st = check_paged(cache, seqs);
  if (st != MI_OK) return st;
  if (n_heads < 0 || n_heads > 65536 || cache->n_kv > 65536)
    return host_fail(MI_ERR_SHAPE, "n_heads=%lld, n_kv=%lld", (long long)n_heads, (long long)cache->n_kv);
  if (rotary && (st = check_rotary(rotary, cache->head_dim)) != MI_OK) return st;
  if (seqs->total_q == 0 || seqs->n_seqs == 0) return MI_OK;
  if (cache->head_dim > ROPE_MAX_DIM)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: at most %d", (long long)cache->head_dim, ROPE_MAX_DIM);
  if (q && !q_out) return host_fail(MI_ERR_NULL, "q_out is NULL");
  if (cache->n_kv > 0 && (!k || !v)) return host_fail(MI_ERR_NULL, "k or v is NULL");
  if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v) % 2)
    return host_fail(MI_ERR_UNSUPPORTED, "pointers must be aligned to their element size");
  const int64_t tokens = seqs->total_q;
  if (q && ((tokens > 1 && qo_t == 0) || (n_heads > 1 && qo_h == 0)))
    return host_fail(MI_ERR_LD, "a stride of q_out is 0: rows would share memory");
  if (q && q == q_out && ((tokens > 1 && q_t != qo_t) || (n_heads > 1 && q_h != qo_h)))
    return host_fail(MI_ERR_UNSUPPORTED, "in place needs the same strides of q and q_out");
  RopeParams p = {};
  int heads[4] = {};
  p.pv = paged_view(cache, seqs);
  if (q && n_heads > 0) {
    p.part[0] = RopePart{q, q_out, 0, q_t, q_h, 0, qo_t, qo_h, 0, rotary != nullptr, 0};
    heads[0] = (int)n_heads;
    p.n_parts = 1;
    p.heads = (int)n_heads;
  }
  if (cache->n_kv > 0 && cache->num_pages > 0) {
    for (int i = 0; i < 2; ++i) {
      p.part[p.n_parts] = RopePart{i ? v : k, i ? cache->v : cache->k, 0, i ? v_t : k_t, i ? v_h : k_h, 0, 0,
                                   cache->head_stride, p.heads, i == 0 && rotary, 1};
      heads[p.n_parts] = (int)cache->n_kv;
      ++p.n_parts;
      p.heads += (int)cache->n_kv;
    }
  }
  if (p.heads == 0) return MI_OK;
  p.d = (int)cache->head_dim;
  p.tokens = p.T = (int)tokens;
  set_rotary(p, rotary, false);
  return rope_run(p, true, true, 1, tokens, heads, stream);
}

}  // extern "C"
