// mi_paged.hip -- attention of a chunk of new tokens over a paged K/V cache, gfx950.
//
// Row (token r, head h) of a sequence with n keys, at position p, reads the keys of KV head
// h / group:  O = sum_j e_j v_j / sum_j e_j,  e_j = exp(scale q.k_j - m),  j <= p (causal) or
// j < n, with the running maximum m and sum of an online softmax in fp32.
//
// A workgroup owns 128 rows of one (sequence, KV head), the group's query heads of a token side by side,
// so one pass over K and V serves all of them; it streams 64-key blocks through a two-stage LDS ring.
// Blocks are gathered row by row from the pages, straight into LDS.  Keys beyond the sequence, in bad
// pages or past head_dim are read from zeros: what a page holds past the sequence may be anything.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "mi_gemm_dlds.hpp"
#include "mi_paged.hpp"

namespace mig {
namespace {

constexpr int PA_ROWS = 128;    // query rows of a workgroup, 32 for each wave
constexpr int PA_KEYS = 64;     // keys of a block
constexpr float PA_TAU = 8.0f;  // growth of a row's maximum (log2 units) that forces a rescale

struct AttnParams {
  PagedView pv;
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  const uint16_t *k, *v;
  float* part_o;    // [pieces][total_q][n_heads][d] normalised outputs of the pieces
  float* part_lse;  // [pieces][total_q][n_heads] log2 of their weight sums
  int64_t q_t, q_h, o_t, o_h;
  int n_heads, n_kv, group, d, causal;
  int tiles;        // row tiles of the launch, some of them empty
  int pieces;       // most pieces that the keys of a tile are cut into
  int min_piece;    // keys of a piece at least
  float scale_log2;
};

// Where rows without a key, and components past head_dim, are read.
__device__ __align__(16) uint32_t pa_zero[4];

// Tile x of the launch: sequence s has the tiles from q_start[s] * group / PA_ROWS + s on, one more than
// it can need, so no prefix sum over the sequences is needed to find a tile's own.
struct PaTile {
  int s, q0, n;   // sequence, its first row and its rows; s < 0: empty
  int first;      // first packed row (token * group + head in group) of the tile
  int64_t len;    // its cached tokens
  int64_t cap;    // what its pages can hold
  __device__ __forceinline__ int64_t limit(const AttnParams& p, int token) const {
    const int64_t e = p.causal ? len - n + token + 1 : len;
    return max((int64_t)0, min(e, cap));
  }
  // keys that the tile's last row sees
  __device__ __forceinline__ int64_t end(const AttnParams& p) const {
    const int64_t last = min((int64_t)first + PA_ROWS, (int64_t)n * p.group) - 1;
    return limit(p, (int)(last / p.group));
  }
};

__device__ __forceinline__ PaTile pa_tile(const AttnParams& p, int x) {
  PaTile t;
  int64_t start;
  if (p.pv.q_start) {
    t.s = wave_first_false(p.pv.n_seqs, [&](int k) {
      const int64_t at = min(max(p.pv.q_start[k + 1], 0), p.pv.total_q);
      return at * p.group / PA_ROWS + k + 1 <= x;
    });
    if (t.s >= p.pv.n_seqs) {
      t.s = -1;
      return t;
    }
    t.s = uniform(t.s);
    seq_rows(p.pv, t.s, t.q0, t.n);
    start = (int64_t)t.q0 * p.group / PA_ROWS + t.s;
  } else {
    const int each = (p.group + PA_ROWS - 1) / PA_ROWS;
    t.s = x / each;
    t.q0 = t.s;
    t.n = 1;
    start = (int64_t)t.s * each;
  }
  const int64_t first = (x - start) * PA_ROWS;
  t.first = (int)first;
  if (first < 0 || first >= (int64_t)t.n * p.group) {
    t.s = -1;
    return t;
  }
  t.q0 = uniform(t.q0);
  t.n = uniform(t.n);
  t.len = uniform(p.pv.kv_len[t.s]);
  t.cap = (int64_t)p.pv.max_pages << p.pv.page_shift;
  return t;
}

// Keys of each piece that [0, end) is cut into, a multiple of PA_KEYS.
__device__ __forceinline__ int64_t pa_piece(const AttnParams& p, int64_t end) {
  const int64_t even = (end + p.pieces - 1) / p.pieces;
  const int64_t len = even > p.min_piece ? even : p.min_piece;
  return (len + PA_KEYS - 1) / PA_KEYS * PA_KEYS;
}

// LDS layout of a 64-key K or V block, rows of D components in 16-byte chunks whose place is XORed with
// bits of the row, so that the 16 rows of a row read, and the 4 rows of a transposing read, lie in
// different banks.
template <int D>
struct PaLds {
  static constexpr int ROW = D * 2;
  static constexpr int NCH = D / 8;
  static constexpr int RPB = 1024 / ROW;          // rows that one 64-lane load brings
  static constexpr int BYTES = PA_KEYS * ROW;
  static constexpr int NU = BYTES / 1024 / 4;     // loads of a wave for a block
  __device__ static __forceinline__ int k_pos(int r, int c) {
    if constexpr (D == 128) return c ^ (r & 15);
    else return c ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
  }
  __device__ static __forceinline__ int v_pos(int r, int c) {
    if constexpr (D == 128) return c ^ ((r & 3) << 2);
    else return c ^ (((r >> 1) & 1) << 2);
  }
};

template <int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) paged_attn_kernel(AttnParams p) {
  using L = PaLds<D>;
  constexpr int NS = D / 16, NC = D / 32, STAGE = 2 * L::BYTES;
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  const uint32_t lds0 = lds_addr(smem);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int h32 = lane >> 5, l32 = lane & 31;

  const int x = uniform(blockIdx.x % p.tiles), rest = uniform(blockIdx.x / p.tiles);
  const int kvh = uniform(rest % p.n_kv), piece = uniform(rest / p.n_kv);
  const PaTile t = pa_tile(p, x);
  if (t.s < 0) return;
  const int64_t end = t.end(p), plen = pa_piece(p, end);
  const int64_t k_begin = piece * plen;
  if (piece > 0 && k_begin >= end) return;
  const int64_t k_end = min(k_begin + plen, end);
  const bool whole = plen >= end;

  // this lane's row; rows past the sequence's last one repeat it and are not stored
  const int n_packed = min(t.n * p.group - t.first, PA_ROWS);
  const bool wave_has_rows = 32 * wave < n_packed;
  const int pr = t.first + min(32 * wave + l32, n_packed - 1);
  const int token = pr / p.group, head = kvh * p.group + pr - token * p.group;
  const int64_t lim = t.limit(p, token);
  // the wave's rows see at least lim_lo and at most lim_hi keys
  const int64_t lim_lo = t.limit(p, (t.first + min(32 * wave, n_packed - 1)) / p.group);
  const int64_t lim_hi = t.limit(p, (t.first + min(32 * wave + 31, n_packed - 1)) / p.group);

  u32x4_t qf[NS];
  {
    const uint16_t* qr = p.q + (t.q0 + token) * p.q_t + head * p.q_h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = 8 * (2 * s + h32);
      qf[s] = c < p.d ? *(const u32x4_t*)(qr + c) : u32x4_t{0, 0, 0, 0};
    }
  }

  // DMA: wave w brings rows 16w .. 16w+15 of a block; in load u lane l brings a chunk of row
  // 16w + RPB*u + l/NCH.
  const uint16_t* kbase = p.k + kvh * p.pv.head_stride;
  const uint16_t* vbase = p.v + kvh * p.pv.head_stride;
  int page_next = -1;   // page of key `lane` of the next block to be issued, read a block ahead of its use
  int64_t row_off = 0;  // element offset of key `lane` of the block issued last, -1: none
  uint64_t seen_next = 0;  // that block's keys that exist
  auto look_up = [&](int64_t base) __attribute__((always_inline)) {
    const int64_t pos = base + lane;
    page_next = pos < k_end ? p.pv.pages[(int64_t)t.s * p.pv.pages_ld + (pos >> p.pv.page_shift)] : -1;
  };
  auto resolve = [&](int64_t base) __attribute__((always_inline)) {
    const bool there = (uint32_t)page_next < (uint32_t)p.pv.num_pages;
    const int slot = (int)(base + lane) & ((1 << p.pv.page_shift) - 1);
    row_off = there ? page_next * p.pv.page_stride + slot * p.pv.slot_stride : -1;
    seen_next = __ballot(there);
  };
  auto issue = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < L::NU; ++u) {
      const int r = 16 * wave + L::RPB * u + lane / L::NCH, at = lane % L::NCH;
      const int64_t off = __shfl(row_off, r, 64);
      const int kc = 8 * L::k_pos(r, at), vc = 8 * L::v_pos(r, at);
      const void* ks = off >= 0 && kc < p.d ? (const void*)(kbase + off + kc) : (const void*)pa_zero;
      const void* vs = off >= 0 && vc < p.d ? (const void*)(vbase + off + vc) : (const void*)pa_zero;
      const uint32_t dst = lds0 + (uint32_t)(stage * STAGE + (wave * L::NU + u) * 1024);
      __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(uintptr_t)ks,
                                       (__attribute__((address_space(3))) void*)(uintptr_t)dst, 16, 0, 0);
      __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(uintptr_t)vs,
                                       (__attribute__((address_space(3))) void*)(uintptr_t)(dst + L::BYTES), 16, 0, 0);
    }
  };

  // the row of a 32-key half that a lane reads: bits 2 and 3 of the key swapped, so that the scores of a
  // lane are, in order, the 8-key runs that the second operand of P V takes
  const int k_row = (l32 & ~0xC) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
  uint32_t v_rd[NC];
  {
    const int g = lane >> 4, jj = lane & 15;
    const int krb = 8 * (g >> 1) + (jj >> 2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = 32 * c + 16 * (g & 1) + 4 * (jj & 3);
      v_rd[c] = (uint32_t)(L::BYTES + krb * L::ROW + 16 * L::v_pos(krb, col >> 3) + (col & 7) * 2);
    }
  }

  f32x16_t o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c][e] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  const float sl2 = p.scale_log2;

  auto block = [&](uint32_t st, uint64_t seen, auto masked) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(masked)::value;
    f32x16_t sc[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[kb][e] = 0.0f;
    u32x4_t kf[NS][2];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        kf[s][kb] = *(const lds_u32x4_t*)(uintptr_t)(st + (uint32_t)((32 * kb + k_row) * L::ROW +
                                                                     16 * L::k_pos(k_row, 2 * s + h32)));
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kf[s][kb]),
                                                        __builtin_bit_cast(bf16x8_t, qf[s]), sc[kb], 0, 0, 0);
    // sc[kb][4q + e] is key 32kb + 8*h32 + 16(q>>1) + 4(q&1) + e
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const uint32_t bits = (uint32_t)(seen >> (32 * kb)) >> (8 * h32);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if constexpr (MASK) {
          const int at = 16 * ((i >> 2) >> 1) + 4 * ((i >> 2) & 1) + (i & 3);
          sc[kb][i] = (bits >> at) & 1 ? sc[kb][i] : -INFINITY;
        }
        mx = fmaxf(mx, sc[kb][i]);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    // a row keeps its reference maximum until a block raises it by more than PA_TAU
    const float m_old = m_run;
    const bool fresh = m_old == -INFINITY, raise = !fresh && (mx - m_old) * sl2 > PA_TAU;
    const float m_ref = fresh || raise ? mx : m_old;
    if (__any(raise)) {
      const float alpha = raise ? __builtin_amdgcn_exp2f((m_old - m_ref) * sl2) : 1.0f;
      l_run *= alpha;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[c][e] *= alpha;
    }
    m_run = m_ref;
    const float nmc = m_ref == -INFINITY ? 0.0f : -m_ref * sl2;
    float sum = 0.0f;
    u32x4_t pf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int kb = ks >> 1, base = 8 * (ks & 1);
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][base + 2 * w2], sl2, nmc));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][base + 2 * w2 + 1], sl2, nmc));
        sum += e0 + e1;
        pf[ks][w2] = pack_bf16x2(e0, e1);
      }
    }
    l_run += sum;
    static_for<4>([&](auto ks_c) __attribute__((always_inline)) {
      constexpr int ks = decltype(ks_c)::value;
      u32x4_t vf[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        static_for<2>([&](auto t_c) __attribute__((always_inline)) {
          constexpr int tt = decltype(t_c)::value;
          u32x2_t w2 = {0u, 0u};
#if defined(__HIP_DEVICE_COMPILE__)
          // inline asm: the builtin would also wait for the loads into LDS that are in flight
          asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"
                       : "=v"(w2)
                       : "v"(st + v_rd[c]), "i"((16 * ks + 4 * tt) * L::ROW));
#endif
          vf[c][2 * tt] = w2[0];
          vf[c][2 * tt + 1] = w2[1];
        });
      }
      // the results are valid after lgkmcnt(0), which the compiler does not know of
      __builtin_amdgcn_s_waitcnt(0xC07F);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                       __builtin_bit_cast(bf16x8_t, pf[ks]), o[c], 0, 0, 0);
    });
  };

  const int n_blocks = uniform((int)((k_end - k_begin + PA_KEYS - 1) / PA_KEYS));
  if (n_blocks > 0) {
    look_up(k_begin);
    resolve(k_begin);
    issue(0);
    look_up(k_begin + PA_KEYS);
  }
  for (int j = 0; j < n_blocks; ++j) {
    const uint64_t seen = seen_next;
    const int64_t base = k_begin + (int64_t)j * PA_KEYS;
    wait_vmcnt<0>();     // this wave's share of block j has landed, and the pages of block j + 1
    lds_ring_barrier();  // and everyone's; and block j - 1 has been read
    if (j + 1 < n_blocks) {
      resolve(base + PA_KEYS);
      issue((j + 1) & 1);
      look_up(base + 2 * PA_KEYS);
    }
    const uint32_t st = lds0 + (uint32_t)((j & 1) * STAGE);
    if (!wave_has_rows || base >= lim_hi) continue;
    if (base + PA_KEYS <= lim_lo && seen == ~uint64_t{0}) {
      block(st, seen, std::false_type{});
    } else {
      const int64_t room = lim - base;
      block(st, room >= 64 ? seen : room <= 0 ? 0 : seen & ((uint64_t{1} << room) - 1), std::true_type{});
    }
  }

  if (!wave_has_rows || 32 * wave + l32 >= n_packed) return;
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
  const int64_t row = t.q0 + token;
  const float lse2 = l_tot == 0.0f ? -INFINITY : m_run * sl2 + __log2f(l_tot);
  if (whole) {
    uint16_t* out = p.o + row * p.o_t + head * p.o_h;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * c + 8 * q < p.d)
          *(u32x2_t*)(out + 32 * c + 8 * q + 4 * h32) =
              u32x2_t{pack_bf16x2(o[c][4 * q] * inv, o[c][4 * q + 1] * inv),
                      pack_bf16x2(o[c][4 * q + 2] * inv, o[c][4 * q + 3] * inv)};
    if (p.lse && h32 == 0) p.lse[row * p.n_heads + head] = lse2 * 0.69314718055994531f;
  } else {
    const int64_t at = ((int64_t)piece * p.pv.total_q + row) * p.n_heads + head;
    float* out = p.part_o + at * p.d;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * c + 8 * q < p.d)
          *(f32x4_t*)(out + 32 * c + 8 * q + 4 * h32) = f32x4_t{o[c][4 * q] * inv, o[c][4 * q + 1] * inv,
                                                                 o[c][4 * q + 2] * inv, o[c][4 * q + 3] * inv};
    if (h32 == 0) p.part_lse[at] = lse2;
  }
}

// Joins the pieces of the rows that have more than one, in their order: o = sum 2^(lse_i - max) o_i over
// the sum of the weights.  One wave a row, two components a lane.
__global__ void __launch_bounds__(256) paged_attn_join_kernel(AttnParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (at >= (int64_t)p.pv.total_q * p.n_heads) return;
  const int row = (int)(at / p.n_heads), head = (int)(at - (int64_t)row * p.n_heads);
  PaTile t;
  t.s = row;
  t.q0 = row;
  t.n = 1;
  if (p.pv.q_start) {
    t.s = wave_first_false(p.pv.n_seqs, [&](int k) { return p.pv.q_start[k + 1] <= row; });
    if (t.s >= p.pv.n_seqs) return;
    seq_rows(p.pv, t.s, t.q0, t.n);
    if (row < t.q0 || row >= t.q0 + t.n) return;
  }
  t.len = p.pv.kv_len[t.s];
  t.cap = (int64_t)p.pv.max_pages << p.pv.page_shift;
  const int packed = (row - t.q0) * p.group + head % p.group;
  t.first = packed / PA_ROWS * PA_ROWS;
  const int64_t end = t.end(p), plen = pa_piece(p, end);
  if (plen >= end) return;
  const int n = (int)((end + plen - 1) / plen);
  const int64_t pitch = (int64_t)p.pv.total_q * p.n_heads;
  float mx = -INFINITY;
  for (int i = lane; i < n; i += 64) mx = fmaxf(mx, p.part_lse[i * pitch + at]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  float sum = 0.0f, a = 0.0f, b = 0.0f;
  for (int i = 0; i < n; ++i) {
    const float li = p.part_lse[i * pitch + at];
    const float w = li == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(li - mx);
    sum += w;
    if (2 * lane < p.d) {
      const float2 x = *(const float2*)(p.part_o + (i * pitch + at) * p.d + 2 * lane);
      a += w * x.x;
      b += w * x.y;
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (2 * lane < p.d) *(uint32_t*)(p.o + row * p.o_t + head * p.o_h + 2 * lane) = pack_bf16x2(a * inv, b * inv);
  if (p.lse && lane == 0)
    p.lse[at] = sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

// Row tiles of a launch, pieces of a tile's keys, and keys of a piece at least.
struct PaPlan {
  int64_t tiles;
  int pieces, min_piece;
  int64_t bytes(int64_t total_q, int64_t n_heads, int64_t d) const {
    return pieces > 1 ? pieces * total_q * n_heads * (d + 1) * 4 : 0;
  }
};

PaPlan pa_plan(int64_t n_heads, int64_t n_kv, int64_t n_seqs, int64_t total_q, int64_t max_q, int64_t max_kv,
               bool one_each, int cus) {
  PaPlan pl;
  const int64_t g = n_heads / n_kv;
  const int64_t per_seq = (std::max<int64_t>(1, std::min(max_q, total_q)) * g + PA_ROWS - 1) / PA_ROWS;
  pl.tiles = one_each ? n_seqs * ((g + PA_ROWS - 1) / PA_ROWS) : n_seqs + total_q * g / PA_ROWS;
  const int64_t units = std::max<int64_t>(1, std::min(pl.tiles, n_seqs * per_seq) * n_kv);
  const int64_t want = (4 * (int64_t)cus + units - 1) / units;
  pl.min_piece = 256;
  const int64_t most = (max_kv + pl.min_piece - 1) / pl.min_piece;
  pl.pieces = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, 256}));
  return pl;
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

size_t mi_paged_attn_workspace_size(int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t n_seqs, int64_t total_q,
                                    int64_t max_q_len, int64_t max_kv_len) {
  if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || head_dim < 1 || n_seqs < 1 || total_q < 1) return 0;
  // CUs of the current device; without one, those of an MI355X
  return (size_t)pa_plan(n_heads, n_kv, n_seqs, total_q, max_q_len, max_kv_len, total_q == n_seqs && max_q_len == 1,
                         host_cus()).bytes(total_q, n_heads, head_dim);
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
  PaPlan plan = pa_plan(n_heads, cache->n_kv, seqs->n_seqs, rows, max_q_len, max_kv_len, !seqs->q_start, host_cus());
  // as many pieces as the workspace holds
  const int64_t piece_bytes = rows * n_heads * (d + 1) * 4;
  if (!workspace) plan.pieces = 1;
  if ((int64_t)workspace_bytes < plan.pieces * piece_bytes)
    plan.pieces = (int)std::max<int64_t>(1, (int64_t)workspace_bytes / piece_bytes);
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
  p.n_kv = (int)cache->n_kv;
  p.causal = causal != 0;
  p.tiles = (int)plan.tiles;
  p.pieces = plan.pieces;
  p.min_piece = plan.min_piece;
  p.part_o = (float*)workspace;
  p.part_lse = p.part_o ? p.part_o + plan.pieces * rows * n_heads * d : nullptr;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int64_t grid = plan.tiles * p.n_kv * plan.pieces;
  if (grid > INT32_MAX) return host_fail(MI_ERR_SHAPE, "too many row tiles");
  if (d <= 64) paged_attn_kernel<64><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(p);
  else paged_attn_kernel<128><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && plan.pieces > 1) {
    paged_attn_join_kernel<<<(unsigned)((rows * n_heads + 3) / 4), 256, 0, (hipStream_t)stream>>>(p);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "paged_attn launch: %s", hipGetErrorString(e));
}

}  // extern "C"
