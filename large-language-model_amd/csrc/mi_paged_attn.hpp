// mi_paged_attn.hpp -- what the attention over a paged cache has in common whatever the cache holds
// (mi_paged.hip: bf16, mi_paged_quant.hip: 8 or 4 bits): tiles of rows, pieces and even shares of the keys, a
// 64-key block of many rows in LDS, the join of few rows' waves, the joins of parts, and the host's plan.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "mi_gemm_dlds.hpp"
#include "mi_paged.hpp"

namespace mig {
namespace {

constexpr int PA_ROWS = 128;    // query rows of a workgroup, 32 for each wave
constexpr int PA_KEYS = 64;     // keys of a block
constexpr int PA_PIECES = 256;  // pieces of a tile's keys at most
constexpr int PF_ROWS = 16;     // the same for few rows: one 16-row tile,
constexpr int PF_KEYS = 32;     // of which every wave takes blocks of its own
constexpr int PF_WAVES = 4;
constexpr int PF_TABLE = 1024;  // entries of the page table that are held in LDS
constexpr float PA_TAU = 8.0f;  // growth of a row's maximum (log2 units) that forces a rescale

struct AttnParams {
  PagedView pv;
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  const void *k, *v;  // of the cache
  float* part_o;    // [pieces][total_q][n_heads][d] normalised outputs of the pieces
  float* part_lse;  // [pieces][total_q][n_heads] log2 of their weight sums
  int64_t q_t, q_h, o_t, o_h;
  int n_heads, n_kv, group, d, causal;
  int tile_shift;   // log2 of the rows of a tile
  int tiles;        // row tiles of the launch, some of them empty
  int pieces;       // most pieces that the keys of a tile are cut into
  int min_piece;    // keys of a piece at least
  int cap;          // keys that a sequence's pages can hold
  int share;        // workgroups of a KV head that share all keys evenly
  uint32_t* prefix; // [n_seqs + 1] blocks of the sequences before each one
  float scale_log2;
};

// Where rows without a key, and components past head_dim, are read.
__device__ __align__(16) uint32_t pa_zero[4];

// Tile x of the launch: sequence s has the tiles from q_start[s] * group / rows + s on, one more than
// it can need, so no prefix sum over the sequences is needed to find a tile's own.
struct PaTile {
  int s, q0, n;   // sequence, its first row and its rows; s < 0: empty
  int first;      // first packed row (token * group + head in group) of the tile
  int len;        // its cached tokens
  __device__ __forceinline__ int limit(const AttnParams& p, int token) const {  // keys that a row sees
    const int64_t e = p.causal ? (int64_t)len - n + token + 1 : len;
    return (int)max((int64_t)0, min(e, (int64_t)p.cap));
  }
  __device__ __forceinline__ int end(const AttnParams& p) const {  // keys that the tile's last row sees
    const int last = min(first + (1 << p.tile_shift), n * p.group) - 1;
    return limit(p, last / p.group);
  }
};

__device__ __forceinline__ PaTile pa_tile(const AttnParams& p, int x) {
  PaTile t;
  int64_t start;
  if (p.pv.q_start) {
    t.s = wave_first_false(p.pv.n_seqs, [&](int k) {
      const int64_t at = min(max(p.pv.q_start[k + 1], 0), p.pv.total_q);
      return (at * p.group >> p.tile_shift) + k + 1 <= x;
    });
    if (t.s >= p.pv.n_seqs) {
      t.s = -1;
      return t;
    }
    t.s = uniform(t.s);
    seq_rows(p.pv, t.s, t.q0, t.n);
    start = ((int64_t)t.q0 * p.group >> p.tile_shift) + t.s;
  } else {
    const int each = (p.group + (1 << p.tile_shift) - 1) >> p.tile_shift;
    t.s = x / each;
    t.q0 = t.s;
    t.n = 1;
    start = (int64_t)t.s * each;
  }
  const int64_t first = (x - start) << p.tile_shift;
  t.first = (int)first;
  if (first < 0 || first >= (int64_t)t.n * p.group) {
    t.s = -1;
    return t;
  }
  t.first = uniform(t.first);
  t.q0 = uniform(t.q0);
  t.n = uniform(t.n);
  t.len = uniform(p.pv.kv_len[t.s]);
  return t;
}

// Keys of each piece that [0, end) is cut into, a multiple of PA_KEYS.
__device__ __forceinline__ int pa_piece(const AttnParams& p, int end) {
  const uint32_t even = ((uint32_t)end + p.pieces - 1) / (uint32_t)p.pieces;
  return (int)((max(even, (uint32_t)p.min_piece) + PA_KEYS - 1) / PA_KEYS * PA_KEYS);
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

__device__ __forceinline__ u32x2_t read_tr16(uint32_t at) {
  typedef short i16x4_t __attribute__((__vector_size__(4 * sizeof(short))));
  typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(uintptr_t)at));
}

// N fragments of V: two transposing reads of 8 bytes each, at[c] + OFF and NEXT bytes further on.  Inline asm: the builtin
// would also wait for the loads into LDS that are in flight.  The wait for all of them ends the asm, so that
// the compiler sees no register before it holds its data.
template <int N, int OFF, int NEXT>
__device__ __forceinline__ void read_v(u32x4_t (&v)[N], uint32_t st, const uint32_t (&at)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "written out for these");
  u32x2_t w[2 * N];
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (N == 2)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
        "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
        : "v"(st + at[0]), "v"(st + at[1]), "i"(OFF), "i"(OFF + NEXT));
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7])
        : "v"(st + at[0]), "v"(st + at[1]), "v"(st + at[2]), "v"(st + at[3]), "i"(OFF), "i"(OFF + NEXT));
  else
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16 offset:%24\n\tds_read_b64_tr_b16 %1, %16 offset:%25\n\t"
        "ds_read_b64_tr_b16 %2, %17 offset:%24\n\tds_read_b64_tr_b16 %3, %17 offset:%25\n\t"
        "ds_read_b64_tr_b16 %4, %18 offset:%24\n\tds_read_b64_tr_b16 %5, %18 offset:%25\n\t"
        "ds_read_b64_tr_b16 %6, %19 offset:%24\n\tds_read_b64_tr_b16 %7, %19 offset:%25\n\t"
        "ds_read_b64_tr_b16 %8, %20 offset:%24\n\tds_read_b64_tr_b16 %9, %20 offset:%25\n\t"
        "ds_read_b64_tr_b16 %10, %21 offset:%24\n\tds_read_b64_tr_b16 %11, %21 offset:%25\n\t"
        "ds_read_b64_tr_b16 %12, %22 offset:%24\n\tds_read_b64_tr_b16 %13, %22 offset:%25\n\t"
        "ds_read_b64_tr_b16 %14, %23 offset:%24\n\tds_read_b64_tr_b16 %15, %23 offset:%25\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7]),
          "=&v"(w[8]), "=&v"(w[9]), "=&v"(w[10]), "=&v"(w[11]), "=&v"(w[12]), "=&v"(w[13]), "=&v"(w[14]), "=&v"(w[15])
        : "v"(st + at[0]), "v"(st + at[1]), "v"(st + at[2]), "v"(st + at[3]), "v"(st + at[4]), "v"(st + at[5]),
          "v"(st + at[6]), "v"(st + at[7]), "i"(OFF), "i"(OFF + NEXT));
#endif
#pragma unroll
  for (int c = 0; c < N; ++c) v[c] = u32x4_t{w[2 * c][0], w[2 * c][1], w[2 * c + 1][0], w[2 * c + 1][1]};
}

// The rows of a wave, 32 of a tile of PA_ROWS, with their running sums.  STREAMED: the blocks come by loads into LDS, which
// are in flight meanwhile, so V's fragments are read in inline asm; else the compiler's reads bring them a step
// ahead, and a wave on a block goes before those that bring the next (16 mixed sequences in 8 bits: neither
// 36.2 us, V ahead 35.6, both 34.5).
template <int D, bool STREAMED>
struct PaRows {
  using L = PaLds<D>;
  static constexpr int NS = D / 16, NC = D / 32;
  int h32, l32;
  int token, head;          // this lane's row; rows past the sequence's last one repeat it and are not stored
  int lim, lim_lo, lim_hi;  // keys that it sees, and that the wave's rows see at least and at most
  int k_row;
  uint32_t v_rd[NC];
  u32x4_t qf[NS];
  f32x16_t o[NC];
  float m_run, l_run, sl2;

  __device__ __forceinline__ void begin(const AttnParams& p, const PaTile& t, int kvh, int wave, int n_packed) {
    const int lane = threadIdx.x & 63;
    h32 = lane >> 5, l32 = lane & 31;
    const int pr = t.first + min(32 * wave + l32, n_packed - 1);
    token = pr / p.group, head = kvh * p.group + pr - token * p.group;
    lim = t.limit(p, token);
    lim_lo = t.limit(p, (t.first + min(32 * wave, n_packed - 1)) / p.group);
    lim_hi = t.limit(p, (t.first + min(32 * wave + 31, n_packed - 1)) / p.group);
    const uint16_t* qr = p.q + (int64_t)(t.q0 + token) * p.q_t + (int64_t)head * p.q_h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = 8 * (2 * s + h32);
      qf[s] = c < p.d ? *(const u32x4_t*)(qr + c) : u32x4_t{0, 0, 0, 0};
    }
    // the row of a 32-key half that a lane reads: bits 2 and 3 of the key swapped, so that the scores of a
    // lane are, in order, the 8-key runs that the second operand of P V takes
    k_row = (l32 & ~0xC) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
    const int g = lane >> 4, jj = lane & 15;
    const int krb = 8 * (g >> 1) + (jj >> 2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = 32 * c + 16 * (g & 1) + 4 * (jj & 3);
      v_rd[c] = (uint32_t)(L::BYTES + krb * L::ROW + 16 * L::v_pos(krb, col >> 3) + (col & 7) * 2);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[c][e] = 0.0f;
    m_run = -INFINITY, l_run = 0.0f;
    sl2 = p.scale_log2;
  }

  __device__ __forceinline__ void fragments(u32x4_t (&v)[NC], uint32_t st) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const u32x2_t a = read_tr16(st + v_rd[c]), b = read_tr16(st + v_rd[c] + 4 * L::ROW);
      v[c] = u32x4_t{a[0], a[1], b[0], b[1]};
    }
  }

  // The 64-key block at LDS address st, K and behind it V, of keys base .. base + 63, of which `seen` exist.
  __device__ __forceinline__ void block(uint32_t st, int base, uint64_t seen) {
    if (base >= lim_hi) return;
    const bool masked = base + PA_KEYS > lim_lo || seen != ~uint64_t{0};
    const int room = lim - base;
    seen = room >= 64 ? seen : room <= 0 ? 0 : seen & ((uint64_t{1} << room) - 1);
    f32x16_t sc[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[kb][e] = 0.0f;
    if constexpr (!STREAMED) __builtin_amdgcn_s_setprio(1);
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
    if (masked) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const uint32_t bits = (uint32_t)(seen >> (32 * kb)) >> (8 * h32);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 16 * ((i >> 2) >> 1) + 4 * ((i >> 2) & 1) + (i & 3);
          sc[kb][i] = (bits >> at) & 1 ? sc[kb][i] : -INFINITY;
        }
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][i]);
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
    u32x4_t hi[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int kb = ks >> 1, base = 8 * (ks & 1);
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][base + 2 * w2], sl2, nmc));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][base + 2 * w2 + 1], sl2, nmc));
        sum += e0 + e1;
        hi[ks][w2] = pack_bf16x2(e0, e1);
        sc[kb][base + 2 * w2] = e0;  // for what hi leaves
        sc[kb][base + 2 * w2 + 1] = e1;
      }
    }
    l_run += sum;
    u32x4_t v[STREAMED ? 1 : 2][NC];
    if constexpr (!STREAMED) fragments(v[0], st);
    static_for<4>([&](auto ks_c) __attribute__((always_inline)) {
      constexpr int ks = decltype(ks_c)::value;
      u32x4_t(&vf)[NC] = v[STREAMED ? 0 : ks & 1];
      u32x4_t lo;
      {
        constexpr int kb = ks >> 1, base = 8 * (ks & 1);
#pragma unroll
        for (int w2 = 0; w2 < 4; ++w2)
          lo[w2] = pack_bf16x2(sc[kb][base + 2 * w2] - bf16_bits_to_f32(hi[ks][w2] & 0xffffu),
                               sc[kb][base + 2 * w2 + 1] - __uint_as_float(hi[ks][w2] & 0xffff0000u));
      }
      if constexpr (STREAMED) {
        read_v<NC, 16 * ks * L::ROW, 4 * L::ROW>(vf, st, v_rd);
        __builtin_amdgcn_sched_barrier(0);
      } else if constexpr (ks < 3) {
        fragments(v[(ks + 1) & 1], st + 16 * (ks + 1) * L::ROW);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                       __builtin_bit_cast(bf16x8_t, lo), o[c], 0, 0, 0);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                       __builtin_bit_cast(bf16x8_t, hi[ks]), o[c], 0, 0, 0);
    });
    if constexpr (!STREAMED) __builtin_amdgcn_s_setprio(0);
  }

  // Writes O and lse, or the part of a piece; bit i of nan(c): component 32c + i of this lane's row is NaN.
  template <class Nan>
  __device__ __forceinline__ void end(const AttnParams& p, const PaTile& t, int wave, int n_packed, int piece,
                                      bool whole, Nan nan) {
    if (32 * wave + l32 >= n_packed) return;
    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
    const int64_t row = t.q0 + token;
    const float lse2 = l_tot == 0.0f ? -INFINITY : m_run * sl2 + __log2f(l_tot);
    if (whole) {
      uint16_t* out = p.o + row * p.o_t + (int64_t)head * p.o_h;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t gone = nan(c) >> (4 * h32);
        auto at = [&](int q, int e) { return o[c][4 * q + e] * ((gone >> (8 * q + e)) & 1 ? NAN : inv); };
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (32 * c + 8 * q < p.d)
            *(u32x2_t*)(out + 32 * c + 8 * q + 4 * h32) =
                u32x2_t{pack_bf16x2(at(q, 0), at(q, 1)), pack_bf16x2(at(q, 2), at(q, 3))};
      }
      if (p.lse && h32 == 0) p.lse[row * p.n_heads + head] = lse2 * 0.69314718055994531f;
    } else {
      const int64_t at = ((int64_t)piece * p.pv.total_q + row) * p.n_heads + head;
      float* out = p.part_o + at * p.d;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const uint32_t gone = nan(c) >> (4 * h32);
        auto at = [&](int q, int e) { return o[c][4 * q + e] * ((gone >> (8 * q + e)) & 1 ? NAN : inv); };
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (32 * c + 8 * q < p.d)
            *(f32x4_t*)(out + 32 * c + 8 * q + 4 * h32) = f32x4_t{at(q, 0), at(q, 1), at(q, 2), at(q, 3)};
      }
      if (h32 == 0) p.part_lse[at] = lse2;
    }
  }
};

// LDS layout of a 32-key block of V of one wave, where rows are few.
template <int D>
struct PfLds {
  static constexpr int ROW = D * 2;
  static constexpr int NCH = D / 8;
  static constexpr int RPB = 1024 / ROW;
  static constexpr int BYTES = PF_KEYS * ROW;
  static constexpr int NU = BYTES / 1024;  // loads for a block of V; as many bring K
  // 16 lanes read 32 bytes of each of four rows of V, the next 16 of the rows 8 further on
  __device__ static __forceinline__ int v_pos(int r, int c) {
    if constexpr (D == 128) return c ^ ((r & 3) << 2) ^ (((r >> 3) & 1) << 1);
    else return c ^ (((r >> 1) & 1) << 2) ^ (((r >> 3) & 1) << 1);
  }
};

template <int D>
constexpr int PF_PITCH = D + 4;  // floats of a row of a wave's sums: its 16-byte stores spread over the banks

// Joins the sums of a workgroup's waves over one tile of few rows: o[c][e] is component 16c + 4g + e of row
// l16, l_run a lane's share of its weights' sum. `ring`: LDS, `pitch` bytes for each wave, with nothing on its way to it.
// O and lse are written if the keys are all of the tile's (whole), else the part at part_at(row, head); bit i of
// nan(token, c): component 32c + i of the token's row is NaN.
struct PfWaves {
  float wm[PF_WAVES][PF_ROWS], wl[PF_WAVES][PF_ROWS];
};
template <int D, class PartAt, class Nan>
__device__ __forceinline__ void pf_join_waves(const AttnParams& p, char* ring, int pitch, PfWaves& lds, const PaTile& t,
                                              int kvh, int n_packed, const f32x4_t (&o)[D / 16], float m_run, float l_run,
                                              bool whole, PartAt part_at, Nan nan) {
  constexpr int ND = D / 16;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
  const float sl2 = p.scale_log2;
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  __syncthreads();
  float* sums = (float*)(ring + wave * pitch);
#pragma unroll
  for (int c = 0; c < ND; ++c) *(f32x4_t*)(sums + l16 * PF_PITCH<D> + 16 * c + 4 * g) = o[c];
  if (g == 0) lds.wm[wave][l16] = m_run, lds.wl[wave][l16] = l_run;
  __syncthreads();
  constexpr int TPR = 64 * PF_WAVES / PF_ROWS;  // threads of a row
  const int r = threadIdx.x / TPR, c0 = threadIdx.x % TPR;
  if (r < n_packed) {
    float m = -INFINITY, l = 0.0f, f[PF_WAVES];
#pragma unroll
    for (int w = 0; w < PF_WAVES; ++w) m = fmaxf(m, lds.wm[w][r]);
#pragma unroll
    for (int w = 0; w < PF_WAVES; ++w) {
      f[w] = lds.wm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((lds.wm[w][r] - m) * sl2);
      l += f[w] * lds.wl[w][r];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int rt = (t.first + r) / p.group, rh = kvh * p.group + t.first + r - rt * p.group;
    const int64_t row = t.q0 + rt;
    const float lse2 = l == 0.0f ? -INFINITY : m * sl2 + __log2f(l);
    const int64_t at = part_at((int)row, rh);
#pragma unroll
    for (int i = 0; i < D / 4 / TPR; ++i) {
      const int c = 4 * (c0 + TPR * i);
      f32x4_t s = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < PF_WAVES; ++w)
        s += f[w] * *(const f32x4_t*)((const float*)(ring + w * pitch) + r * PF_PITCH<D> + c);
      if (c >= p.d) continue;
      const uint32_t gone = nan(rt, c / 32) >> (c % 32);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] *= (gone >> e) & 1 ? NAN : inv;
      if (whole)
        *(u32x2_t*)(p.o + row * p.o_t + (int64_t)rh * p.o_h + c) = u32x2_t{pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
      else
        *(f32x4_t*)(p.part_o + at * p.d + c) = s;
    }
    if (c0 == 0) {
      if (!whole) p.part_lse[at] = lse2;
      else if (p.lse) p.lse[row * p.n_heads + rh] = lse2 * 0.69314718055994531f;
    }
  }
}

// The sequence of a row (s < 0: none), and the pieces of the keys of one of its heads' tile.
__device__ __forceinline__ PaTile pa_row_tile(const AttnParams& p, int row) {
  PaTile t;
  t.s = row;
  t.q0 = row;
  t.n = 1;
  if (p.pv.q_start) {
    t.s = wave_first_false(p.pv.n_seqs, [&](int k) { return p.pv.q_start[k + 1] <= row; });
    if (t.s < p.pv.n_seqs) seq_rows(p.pv, t.s, t.q0, t.n);
    if (t.s >= p.pv.n_seqs || row < t.q0 || row >= t.q0 + t.n) {
      t.s = -1;
      return t;
    }
  }
  t.len = p.pv.kv_len[t.s];
  return t;
}
__device__ __forceinline__ int pa_pieces_of(const AttnParams& p, PaTile t, int row, int head) {
  const int packed = (row - t.q0) * p.group + head % p.group;
  t.first = packed >> p.tile_shift << p.tile_shift;
  const int end = t.end(p), plen = pa_piece(p, end);
  return plen >= end ? 1 : (int)(((uint32_t)end + plen - 1) / (uint32_t)plen);
}

// One new token for each sequence: the keys of all sequences, in blocks of PF_BLOCK, are one line that the
// workgroups of a KV head share evenly, so that sequences of any lengths keep all CUs busy to the end
// (64 sequences of 500 to 8000 keys, 372 MB: 78 us, in pieces 88 at best).  A workgroup's share lies
// in one sequence or runs over several; only its first and its last may be cut.
constexpr int PF_BLOCK = PF_KEYS * PF_WAVES;
constexpr int PF_SEQS = 1024;   // sequences whose lengths a workgroup sums up
constexpr int PF_SHARES = 1024;  // shares of a KV head, all of which one sequence may be cut into

// First block of workgroup w's share of n blocks.
__device__ __forceinline__ uint32_t pf_share(uint32_t n, uint32_t w, uint32_t of) {
  const uint32_t q = n / of;
  return w * q + min(w, n - q * of);
}
// The workgroup whose share block b is in.
__device__ __forceinline__ uint32_t pf_owner(uint32_t n, uint32_t b, uint32_t of) {
  const uint32_t q = n / of, longer = n - q * of, cut = longer * (q + 1);
  return b < cut ? b / (q + 1) : longer + (b - cut) / q;
}

struct PfPrefix {
  uint32_t prefix[PF_SEQS + 1], wave_sum[PF_WAVES];
};

// Workgroup w of KV head kvh over its share: segment(tile, first key, last key, whole, part_at) for each sequence
// in it, all threads together.  A sequence's keys come after EXTRA blocks of none, for what a workgroup spends on going
// over to it; a share that ends among these has none of its keys.
template <int EXTRA, class Segment>
__device__ __forceinline__ void pf_over_share(const AttnParams& p, PfPrefix& lds, uint32_t w, Segment segment) {
  uint32_t* prefix = lds.prefix;
  uint32_t* wave_sum = lds.wave_sum;
  const int tid = threadIdx.x, lane = tid & 63, S = p.pv.n_seqs;
  constexpr int EACH = PF_SEQS / (64 * PF_WAVES);
  uint32_t n[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = EACH * tid + i;
    n[i] = s < S ? (uint32_t)(min(max(p.pv.kv_len[s], 0), p.cap) + PF_BLOCK - 1) / PF_BLOCK : 0;
    n[i] += n[i] ? EXTRA : 0;
    sum += n[i];
  }
  uint32_t before = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = (uint32_t)__shfl_up((int)before, o, 64);
    if (lane >= o) before += y;
  }
  if (lane == 63) wave_sum[tid >> 6] = before;
  __syncthreads();
  before -= sum;
#pragma unroll
  for (int i = 0; i < PF_WAVES; ++i) before += i < tid >> 6 ? wave_sum[i] : 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = EACH * tid + i;
    if (s <= S) prefix[s] = before;
    before += n[i];
  }
  if (tid == 64 * PF_WAVES - 1 && S == PF_SEQS) prefix[S] = before;
  __syncthreads();
  if (blockIdx.x == 0)  // for the join
    for (int s = tid; s <= S; s += 64 * PF_WAVES) p.prefix[s] = prefix[s];

  const uint32_t total = uniform((int)prefix[S]);
  uint32_t b = pf_share(total, w, p.share);
  const uint32_t stop = pf_share(total, w + 1, p.share);
  if (b >= stop) return;
  int s = uniform(wave_first_false(S, [&](int k) { return prefix[k + 1] <= b; }));
  for (int k = 0; b < stop; k = 1, ++s) {
    const uint32_t first = uniform((int)prefix[s]), next = uniform((int)prefix[s + 1]);
    if (next <= b) continue;
    PaTile t;
    t.s = t.q0 = s;
    t.n = 1;
    t.first = 0;
    t.len = uniform(p.pv.kv_len[s]);
    const int len = t.limit(p, 0);
    const uint32_t last = min(stop, next);
    const int k_begin = max((int)(b - first) - EXTRA, 0) * PF_BLOCK;
    const int k_end = last == next ? len : max((int)(last - first) - EXTRA, 0) * PF_BLOCK;
    segment(t, k_begin, k_end, b == first && last == next,
            [&](int, int head) { return (int64_t)(2 * w + k) * p.n_heads + head; });
    b = last;
    if (b < stop) __syncthreads();  // the waves' sums have been read
  }
}

// Joins n parts of one row, part i at at(i): o = sum 2^(lse_i - max) o_i over the sum of the weights.  A
// workgroup: 32 lanes read a part's components, eight parts at a time and eight such in flight; their sums
// are joined in a fixed order.
template <int MOST, class At>  // n <= MOST
__device__ __forceinline__ void pa_join(const AttnParams& p, int64_t row, int head, int n, At at) {
  __shared__ f32x4_t part[8][32];
  __shared__ float weight[MOST], wave_max[4], slice_sum[8];
  const int tid = threadIdx.x, slice = tid >> 5, l32 = tid & 31;
  float mine[MOST / 256], mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < MOST / 256; ++j) {
    mine[j] = tid + 256 * j < n ? p.part_lse[at(tid + 256 * j)] : -INFINITY;
    mx = fmaxf(mx, mine[j]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if ((tid & 63) == 0) wave_max[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
#pragma unroll
  for (int j = 0; j < MOST / 256; ++j)
    weight[tid + 256 * j] = mine[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine[j] - mx);
  __syncthreads();
  const int c = 4 * l32;
  f32x4_t acc = {0, 0, 0, 0};
  float sum = 0.0f;
  if (c < p.d) {
#pragma unroll 8
    for (int i = slice; i < n; i += 8) {
      sum += weight[i];
      acc += weight[i] * *(const f32x4_t*)(p.part_o + at(i) * p.d + c);
    }
  }
  part[slice][l32] = acc;
  if (l32 == 0) slice_sum[slice] = sum;
  __syncthreads();
  if (slice > 0) return;
  sum = 0.0f;
  acc = f32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum += slice_sum[i];
    acc += part[i][l32];
  }
  acc *= sum == 0.0f ? 0.0f : 1.0f / sum;
  if (c < p.d)
    *(u32x2_t*)(p.o + row * p.o_t + (int64_t)head * p.o_h + c) =
        u32x2_t{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
  if (p.lse && l32 == 0)
    p.lse[row * p.n_heads + head] = sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

// The shares of the sequences that are cut, and the rows of those without a key.
__global__ void __launch_bounds__(256) paged_attn_share_join_kernel(AttnParams p) {
  const int s = (int)(blockIdx.x / p.n_heads), head = (int)(blockIdx.x - (uint32_t)s * p.n_heads);
  const uint32_t total = p.prefix[p.pv.n_seqs], first = p.prefix[s], next = p.prefix[s + 1];
  uint32_t w0 = 0;
  int n = 0, k0 = 0;
  if (next > first) {
    w0 = pf_owner(total, first, p.share);
    n = (int)(pf_owner(total, next - 1, p.share) - w0) + 1;
    if (n == 1) return;
    k0 = pf_share(total, w0, p.share) != first;  // its last one, not its first
  }
  pa_join<PF_SHARES>(p, s, head, n, [&](int i) { return (int64_t)(2 * (w0 + i) + (i == 0 ? k0 : 0)) * p.n_heads + head; });
}

// The pieces of the rows that have more than one: a workgroup a row.
__global__ void __launch_bounds__(256) paged_attn_join_kernel(AttnParams p) {
  const int64_t at = blockIdx.x;
  const int row = (int)(at / p.n_heads), head = (int)(at - (int64_t)row * p.n_heads);
  const PaTile t = pa_row_tile(p, row);
  if (t.s < 0) return;
  const int n = pa_pieces_of(p, t, row, head);
  if (n < 2) return;
  const int64_t pitch = (int64_t)p.pv.total_q * p.n_heads;
  pa_join<PA_PIECES>(p, row, head, n, [&](int i) { return i * pitch + at; });
}

// The same for up to eight pieces of many rows: 32 lanes a head, eight heads of a token a workgroup, all
// pieces' loads in flight.
__global__ void __launch_bounds__(256) paged_attn_join8_kernel(AttnParams p) {
  const int each = (p.n_heads + 7) >> 3, row = uniform(blockIdx.x / each);
  const int l32 = threadIdx.x & 31, c = 4 * l32, head = 8 * (int)(blockIdx.x - row * each) + (threadIdx.x >> 5);
  const PaTile t = pa_row_tile(p, row);
  if (t.s < 0 || head >= p.n_heads) return;
  const int64_t pitch = (int64_t)p.pv.total_q * p.n_heads;
  const int n = pa_pieces_of(p, t, row, head);
  if (n < 2) return;
  const int64_t at = (int64_t)row * p.n_heads + head;
  float lse[8];
  f32x4_t x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lse[i] = i < n ? p.part_lse[i * pitch + at] : -INFINITY;
    x[i] = i < n && c < p.d ? *(const f32x4_t*)(p.part_o + (i * pitch + at) * p.d + c) : f32x4_t{0, 0, 0, 0};
  }
  float mx = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = fmaxf(mx, lse[i]);
  f32x4_t acc = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = lse[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lse[i] - mx);
    sum += w;
    acc += w * x[i];
  }
  acc *= sum == 0.0f ? 0.0f : 1.0f / sum;
  if (c < p.d)
    *(u32x2_t*)(p.o + (int64_t)row * p.o_t + (int64_t)head * p.o_h + c) =
        u32x2_t{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
  if (p.lse && l32 == 0) p.lse[at] = sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

// How a launch is laid out: tiles of rows, pieces of a tile's keys, and keys of a piece at least.
struct PaPlan {
  bool few;
  int share;  // workgroups of a KV head that share the keys evenly, 0: pieces
  int tile_shift;
  int64_t tiles;
  int pieces, min_piece;
  int64_t bytes(int64_t total_q, int64_t n_heads, int64_t d) const {
    return pieces > 1 ? pieces * total_q * n_heads * (d + 1) * 4 : 0;
  }
  int64_t share_bytes(int64_t n_seqs, int64_t n_heads, int64_t d) const {
    return share ? 2 * (int64_t)share * n_heads * (d + 1) * 4 + (n_seqs + 1) * 4 : 0;
  }
};

// Decode (graph replays, us; 16 / 4 heads of 128): one piece up to 512 keys (256 keys 8.6, in two pieces
// and a join 10.5; 512 alike, 10.8 and 10.6 in four); else a workgroup for each CU, of 128 keys at least (one
// sequence of 32768: 22.4, in twice as many pieces 25.4; of 2048: 11.0, in half as many 12.2).
// Even shares instead where the sequences are several and long, 1024 keys a piece and 2048 at least. Lengths that
// differ gain (lengths up to the one given, pieces / shares), alike ones lose less than that:
//    sequences x keys   64 x 1500    64 x 2000    64 x 8000   256 x 1500  256 x 2000  16 x 4000    16 x 8000
//              uneven   23.8/23.7    29.2/27.1   103.4/61.8   51.8/57.1   77.2/78.9   22.3/22.8    33.0/28.5
//                even   34.0/39.3    43.1/47.8   180.0/188    137/142     179/185     28.7/29.9    45.6/49.1
// Many rows: pieces of 512 keys at least until there are two workgroups for each CU, which fit at once; four
// where the sequences are eight or more, of which some are short. With two / four, uneven lengths and even:
//    sequences: rows/keys  6: 64/6000  8: 64/6000  32: 64/6000  6: 700/1400  10: 700/1400  4: 1024/4095  10: 1024/4095
//                 uneven   39.6/38.5   39.5/38.0   83.7/64.0    38.6/38.9    45.4/39.4     75.3/81.0     109.8/97.7
//                   even   59.5/63.4   68.9/71.2   228.7/203.9  77.7/92.8    109.3/140.4   182.8/196.4   449.3/449.7
// Where that leaves CUs empty, pieces of 256 or 128 keys. One sequence, rows over keys, with 128 / 256 / 512:
// 8 over 4000 13.1/15.1/21.0, 17 over 2000 13.6/16.1/22.5 (128 taken), 64 over 4000 26.4/22.1/24.9 (128 taken, 4 us
// too many), 4 sequences of 64 over 2000 32.9/27.3/26.4 (256 taken).
PaPlan pa_plan(int64_t n_heads, int64_t n_kv, int64_t d, int64_t n_seqs, int64_t total_q, int64_t max_q, int64_t max_kv,
               bool one_each, int cus) {
  PaPlan pl;
  const int64_t g = n_heads / n_kv, q = std::max<int64_t>(1, std::min(max_q, total_q));
  max_kv = std::min<int64_t>(max_kv, INT32_MAX);
  pl.few = q * g <= PF_ROWS;
  pl.tile_shift = pl.few ? 4 : 7;
  const int64_t rows = int64_t{1} << pl.tile_shift;
  pl.tiles = one_each ? n_seqs * ((g + rows - 1) / rows) : n_seqs + total_q * g / rows;
  const int64_t units = std::max<int64_t>(1, std::min(pl.tiles, n_seqs * ((q * g + rows - 1) / rows)) * n_kv);
  const int64_t want = ((pl.few ? 1 : n_seqs < 8 ? 2 : 4) * (int64_t)cus + units - 1) / units;
  pl.min_piece = pl.few ? (max_kv <= 512 ? 512 : 128) : 512;
  if (!pl.few && units * ((max_kv + 511) / 512) <= cus) pl.min_piece = units * ((max_kv + 255) / 256) <= cus / 2 ? 128 : 256;
  const int64_t most = (max_kv + pl.min_piece - 1) / pl.min_piece;
  pl.pieces = (int)std::max<int64_t>(1, std::min<int64_t>({want, most, PA_PIECES}));
  // two workgroups on a CU, three of 64 components
  pl.share = one_each && g <= PF_ROWS && n_seqs > 1 && n_seqs <= PF_SEQS && max_kv > 1024 * (int64_t)std::max(pl.pieces, 2)
                 ? (int)std::max<int64_t>(1, std::min<int64_t>((d <= 64 ? 3 : 2) * (int64_t)cus / n_kv, PF_SHARES))
                 : 0;
  // The joins have a workgroup for each row and head.  Only a max_q_len far below the sequences' rows cuts so many.
  if (total_q * n_heads > host_most_groups(256)) pl.pieces = 1, pl.share = 0;
  return pl;
}

// Looks over the arguments of an attention call and fills in p and plan; launch: whether there is anything to do.
// p.share is set where the keys are shared evenly; p.k and p.v are left to the caller.
inline int pa_prepare(AttnParams& p, PaPlan& plan, bool& launch, const void* Q, int64_t q_t, int64_t q_h, void* O, int64_t o_t,
                      int64_t o_h, float* lse, int64_t n_heads, int64_t n_kv, int64_t d, int64_t page_size,
                      const mi_paged_seqs* seqs, const PagedView& view, int64_t max_q_len, int64_t max_kv_len, int32_t causal,
                      float scale, void* workspace, size_t workspace_bytes) {
  launch = false;
  if (n_heads < 0 || max_q_len < 0 || max_kv_len < 0) return host_fail(MI_ERR_SHAPE, "negative size");
  if (seqs->n_seqs == 0 || seqs->total_q == 0 || n_heads == 0) return MI_OK;
  if (n_kv < 1 || n_heads % n_kv || n_heads > 65536)
    return host_fail(MI_ERR_SHAPE, "n_heads=%lld is no multiple of n_kv=%lld", (long long)n_heads,
                     (long long)n_kv);
  if (d > 128)
    return host_fail(MI_ERR_UNSUPPORTED, "head_dim %lld: at most 128", (long long)d);
  if (!Q || !O) return host_fail(MI_ERR_NULL, "Q or O is NULL");
  if (((uintptr_t)Q | (uintptr_t)O | (uintptr_t)workspace) & 15)
    return host_fail(MI_ERR_UNSUPPORTED, "Q, O and the workspace must be 16-byte aligned");
  if ((uintptr_t)lse & 3) return host_fail(MI_ERR_UNSUPPORTED, "lse must be aligned to its element size");
  if ((q_t | q_h | o_t | o_h) % 8) return host_fail(MI_ERR_UNSUPPORTED, "strides of Q and O must be multiples of 8");
  const int64_t rows = seqs->total_q;
  if ((rows > 1 && (o_t < d || q_t < 0)) || (n_heads > 1 && (o_h < d || q_h < 0)))
    return host_fail(MI_ERR_LD, "a stride of O is shorter than a row of %lld", (long long)d);
  if (Q == O && ((rows > 1 && q_t != o_t) || (n_heads > 1 && q_h != o_h)))
    return host_fail(MI_ERR_UNSUPPORTED, "in place needs the same strides of Q and O");
  if (!(scale > 0.0f) || !isfinite(scale * 1.4426950408889634f))
    return host_fail(MI_ERR_UNSUPPORTED, "scale must be positive and finite");
  if (rows * n_heads > INT32_MAX) return host_fail(MI_ERR_SHAPE, "total_q * n_heads exceeds 2^31-1");
  const int st = host_device();
  if (st != MI_OK) return st;
  plan = pa_plan(n_heads, n_kv, d, seqs->n_seqs, rows, max_q_len, max_kv_len, !seqs->q_start, host_cus());
  if (seqs->n_seqs * (seqs->max_pages * page_size / PF_BLOCK + 1) > INT32_MAX) plan.share = 0;  // its sums
  // as many pieces as the workspace holds
  const int64_t piece_bytes = rows * n_heads * (d + 1) * 4;
  if (!workspace) plan.pieces = 1;
  if ((int64_t)workspace_bytes < plan.pieces * piece_bytes)
    plan.pieces = (int)std::max<int64_t>(1, (int64_t)workspace_bytes / piece_bytes);
  p.pv = view;
  p.q = (const uint16_t*)Q;
  p.o = (uint16_t*)O;
  p.lse = lse;
  p.q_t = q_t, p.q_h = q_h, p.o_t = o_t, p.o_h = o_h;
  p.n_heads = (int)n_heads;
  p.group = (int)(n_heads / n_kv);
  p.d = (int)d;
  p.n_kv = (int)n_kv;
  p.causal = causal != 0;
  p.tile_shift = plan.tile_shift;
  p.tiles = (int)plan.tiles;
  p.pieces = plan.pieces;
  p.min_piece = plan.min_piece;
  p.cap = (int)(seqs->max_pages * page_size);
  p.part_o = (float*)workspace;
  p.part_lse = p.part_o ? p.part_o + plan.pieces * rows * n_heads * d : nullptr;
  p.share = 0;
  p.prefix = nullptr;
  p.scale_log2 = scale * 1.4426950408889634f;
  if (plan.share && workspace && plan.share_bytes(rows, n_heads, d) <= (int64_t)workspace_bytes) {
    p.share = plan.share;
    p.part_lse = p.part_o + 2 * (int64_t)p.share * n_heads * d;
    p.prefix = (uint32_t*)(p.part_lse + 2 * (int64_t)p.share * n_heads);
  }
  launch = true;
  return MI_OK;
}

// Launches share(workgroups), few(workgroups) or many(workgroups), and the join of what they leave in parts.
template <class Share, class Few, class Many>
inline int pa_launch(const AttnParams& p, const PaPlan& plan, hipStream_t stream, Share share, Few few, Many many) {
  const int64_t rows = p.pv.total_q, n_heads = p.n_heads;
  hipError_t e;
  if (p.share) {
    share((unsigned)(p.share * p.n_kv));
    e = hipGetLastError();
    if (e == hipSuccess) {
      paged_attn_share_join_kernel<<<(unsigned)(rows * n_heads), 256, 0, stream>>>(p);
      e = hipGetLastError();
    }
    return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "paged_attn launch: %s", hipGetErrorString(e));
  }
  const int64_t grid = plan.tiles * p.n_kv * plan.pieces, most = host_most_groups(256);
  if (grid > most)
    return host_fail(MI_ERR_SHAPE, "%lld row tiles of %lld KV heads: more than %lld workgroups", (long long)plan.tiles,
                     (long long)p.n_kv, (long long)most);
  if (plan.few) few((unsigned)grid);
  else many((unsigned)grid);
  e = hipGetLastError();
  if (e == hipSuccess && plan.pieces > 1) {
    const unsigned wgs8 = (unsigned)(rows * ((n_heads + 7) / 8));
    if (plan.pieces <= 8 && !plan.few) paged_attn_join8_kernel<<<wgs8, 256, 0, stream>>>(p);
    else paged_attn_join_kernel<<<(unsigned)(rows * n_heads), 256, 0, stream>>>(p);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "paged_attn launch: %s", hipGetErrorString(e));
}

// Bytes of the parts that a call with these sizes makes.
inline size_t pa_workspace_size(int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t n_seqs, int64_t total_q,
                                int64_t max_q_len, int64_t max_kv_len) {
  if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || head_dim < 1 || n_seqs < 1 || total_q < 1) return 0;
  if (n_seqs > INT32_MAX || total_q > INT32_MAX / n_heads) return 0;  // refused by the call
  // CUs of the current device, whose table the first of all calls fills in; without one, those of an MI355X
  const int cus = host_device() == MI_OK ? host_cus() : 256;
  const PaPlan plan = pa_plan(n_heads, n_kv, head_dim, n_seqs, total_q, max_q_len, max_kv_len,
                              total_q == n_seqs && max_q_len == 1, cus);
  return (size_t)std::max(plan.bytes(total_q, n_heads, head_dim), plan.share_bytes(n_seqs, n_heads, head_dim));
}

}  // namespace
}  // namespace mig
