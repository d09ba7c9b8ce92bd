// mi_paged.hip -- attention of a chunk of new tokens over a paged K/V cache, gfx950.
//
// Row (token r, head h) of a sequence with n keys, at position p, reads the keys of KV head
// h / group:  O = sum_j e_j v_j / sum_j e_j,  e_j = exp(scale q.k_j - m),  j <= p (causal) or
// j < n, with the running maximum m and sum of an online softmax in fp32.
//
// Bound by reading the keys once for a KV head's group where rows are few, by the matrix cores where they
// are many.  Few rows (decode) have kernels of their own below: 64 sequences of up to 8000 keys, 372 MB in
// 78 us (4.8 TB/s; equal lengths reach 5.3 to 5.9, plain reads 6.0); one of 2048 keys takes 11 us, two
// launches.  Many: 4096 rows over 8192 keys in 317 us (650 TFLOP/s of the formula's operations, half as many
// again are done), 4 chunks of up to 1024 rows over 4095 in 73 (420).  There the matrix cores are busy for 53 and
// 44 % of the busy CUs' clocks, LDS for 18 and 15 %, and waits for LDS are 3 and 2 % of the waves' cycles: what is
// left is each wave's chain of product, maximum, exponentials and product, with two waves on a SIMD to hide it.
// Computing the next block's scores under the exponentials instead only took registers (66 -> 72 us).
//
// A workgroup owns 128 rows of one (sequence, KV head), the group's query heads of a token side by side,
// so one pass over K and V serves all of them; it streams 64-key blocks through a two-stage LDS ring.
// P goes into its product with V as the sum of two bf16, in every kernel: what is left out is 2^-16 of a weight,
// so an output is as exact as its own rounding, whichever rows share its tile.  Many rows pay 21 % for the second
// product (4 chunks of up to 1024 rows over 4095 keys) and 29 % (4096 over 8192); with one bf16 their outputs were
// off by up to 2^-8 of sum p |v| more than those of decode.
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
  const uint16_t *k, *v;
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

// N fragments of V: two transposing reads of 8 bytes each, at[c] + OFF and 4 rows further on.  Inline asm: the builtin
// would also wait for the loads into LDS that are in flight.  The wait for all of them ends the asm, so that
// the compiler sees no register before it holds its data.
template <int N, int OFF, int ROW>
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
        : "v"(st + at[0]), "v"(st + at[1]), "i"(OFF), "i"(OFF + 4 * ROW));
  else if constexpr (N == 4)
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7])
        : "v"(st + at[0]), "v"(st + at[1]), "v"(st + at[2]), "v"(st + at[3]), "i"(OFF), "i"(OFF + 4 * ROW));
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
          "v"(st + at[6]), "v"(st + at[7]), "i"(OFF), "i"(OFF + 4 * ROW));
#endif
#pragma unroll
  for (int c = 0; c < N; ++c) v[c] = u32x4_t{w[2 * c][0], w[2 * c][1], w[2 * c + 1][0], w[2 * c + 1][1]};
}

// Few rows (decode): 16 rows of one (sequence, KV head) for a workgroup, bound by the keys and values that
// it streams.  Every wave takes 32-key blocks of its own, so nothing waits at a barrier until the waves'
// sums are joined at the end: K of the next block comes into registers, where the product wants it, V of
// the next two into an LDS ring of the wave's own.  With eight waves on a CU 128 KB or more are on their way
// to it at any time.
//   S = K Q^T on v_mfma_f32_16x16x32_bf16: lane l holds row l % 16 and, in the two 16-key tiles t, the keys
//   8 (l / 16) + 4t + e: tile t's row r reads key 8 (r / 4) + 4t + r % 4, so that these eight are, in order,
//   the run of keys that the second operand of P V takes.
// The second bf16 of P costs nothing here.
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
struct PfShared {
  __attribute__((aligned(16))) char ring[PF_WAVES * 2 * PfLds<D>::BYTES];
  int table[PF_TABLE];
  float wm[PF_WAVES][PF_ROWS], wl[PF_WAVES][PF_ROWS];
};

// Keys [k_begin, k_end) of a tile of KV head kvh; whole: they are all its keys, and O and lse are written;
// else the part, at part_at(row of the sequence, head).
template <int D, class PartAt>
__device__ __forceinline__ void pf_segment(const AttnParams& p, PfShared<D>& lds, const PaTile& t, int kvh,
                                           int k_begin, int k_end, bool whole, PartAt part_at) {
  using L = PfLds<D>;
  constexpr int NS = D / 32, ND = D / 16, NU = L::NU;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int g = lane >> 4, l16 = lane & 15;
  const uint32_t ring = lds_addr(lds.ring) + (uint32_t)(wave * 2 * L::BYTES);

  const int n_packed = min(t.n * p.group - t.first, PF_ROWS);
  const int pr = t.first + min(l16, n_packed - 1);
  const int token = pr / p.group, head = kvh * p.group + pr - token * p.group;
  const int lim = t.limit(p, token), lim_lo = t.limit(p, t.first / p.group);

  u32x4_t qf[NS];
  {
    const uint16_t* qr = p.q + (int64_t)(t.q0 + token) * p.q_t + (int64_t)head * p.q_h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = 32 * s + 8 * g;
      qf[s] = c < p.d ? *(const u32x4_t*)(qr + c) : u32x4_t{0, 0, 0, 0};
    }
  }

  const uint16_t* kbase = p.k + (int64_t)kvh * p.pv.head_stride;
  const uint16_t* vbase = p.v + (int64_t)kvh * p.pv.head_stride;
  const int shift = p.pv.page_shift;
  const int64_t slot_stride = p.pv.slot_stride;
  // The keys' pages, from first_page on, lie in LDS: a look-up in memory for each block would wait for the
  // keys asked for before it.
  int first_page = 0, k_stop = 0;  // the table holds the pages of the keys before k_stop

  // This lane's K rows of a block (8 (l16 / 4) + l16 % 4, and 4 more), chunks 4s + g; its V rows of the
  // loads u (RPB*u + lane / NCH), and the chunk whose place it fills.
  const int k_row = 8 * (l16 >> 2) + (l16 & 3);
  const uint16_t* k_at[2];  // of the block resolved last
  uint32_t seen;            // its keys that exist
  // whole blocks whose halves lie in one page each: scalar bases and these offsets
  const bool even = shift >= 4 && p.d == D && slot_stride <= (1 << 24);
  uint32_t k_off[2], v_off[NU];
#pragma unroll
  for (int i = 0; i < 2; ++i) k_off[i] = (uint32_t)(((k_row + 4 * i) & 15) * slot_stride + 8 * g);
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int r = L::RPB * u + lane / L::NCH;
    v_off[u] = (uint32_t)((r & 15) * slot_stride + 8 * L::v_pos(r, lane % L::NCH));
  }
  auto to_lds = [&](const uint16_t* src, uint32_t dst) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(uintptr_t)src,
                                     (__attribute__((address_space(3))) void*)(uintptr_t)dst, 16, 0, 0);
  };
  // Asks for V of the block at `base` and notes where its K lies.  A block past the end is asked for from
  // zeros, so that every step has the same loads on their way.
  auto fetch = [&](int base, int stage) __attribute__((always_inline)) {
    const uint32_t dst = ring + (uint32_t)(stage * L::BYTES);
    const int last = k_stop - 1;
    const int p0 = uniform(lds.table[(min(base, last) >> shift) - first_page]);
    const int p1 = uniform(lds.table[(min(base + PF_KEYS - 1, last) >> shift) - first_page]);
    if (even && base + PF_KEYS <= k_stop && (uint32_t)p0 < (uint32_t)p.pv.num_pages &&
        (uint32_t)p1 < (uint32_t)p.pv.num_pages) {
      const int mask = (1 << shift) - 1;
      const int64_t h0 = p0 * p.pv.page_stride + (base & mask) * slot_stride;
      const int64_t h1 = p1 * p.pv.page_stride + ((base + 16) & mask) * slot_stride;
      const int64_t hk = l16 >= 8 ? h1 : h0;
#pragma unroll
      for (int i = 0; i < 2; ++i) k_at[i] = kbase + hk + k_off[i];
#pragma unroll
      for (int u = 0; u < NU; ++u) to_lds(vbase + (u < NU / 2 ? h0 : h1) + v_off[u], dst + u * 1024);
      seen = ~0u;
    } else {
      const int pos = base + (lane & 31);
      const int page = lds.table[(min(pos, last) >> shift) - first_page];
      const bool there = pos < k_stop && (uint32_t)page < (uint32_t)p.pv.num_pages;
      const int64_t off = there ? page * p.pv.page_stride + (pos & ((1 << shift) - 1)) * slot_stride : -1;
      seen = (uint32_t)__ballot(there);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t o = __shfl(off, k_row + 4 * i, 64);
        k_at[i] = o >= 0 ? kbase + o + 8 * g : nullptr;
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int r = L::RPB * u + lane / L::NCH, c = 8 * L::v_pos(r, lane % L::NCH);
        const int64_t o = __shfl(off, r, 64);
        to_lds(o >= 0 && c < p.d ? vbase + o + c : (const uint16_t*)pa_zero, dst + u * 1024);
      }
    }
  };
  u32x4_t kf[NS][2];
  auto fetch_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        kf[s][i] = *(const u32x4_t*)(k_at[i] && 32 * s + 8 * g < p.d ? k_at[i] + 32 * s : (const uint16_t*)pa_zero);
  };

  uint32_t v_rd[ND];
#pragma unroll
  for (int c = 0; c < ND; ++c) {
    const int r = 8 * g + (l16 >> 2), col = 16 * c + 4 * (l16 & 3);
    v_rd[c] = (uint32_t)(r * L::ROW + 16 * L::v_pos(r, col >> 3) + (col & 7) * 2);
  }

  f32x4_t o[ND];
#pragma unroll
  for (int c = 0; c < ND; ++c) o[c] = f32x4_t{0, 0, 0, 0};
  float m_run = -INFINITY, l_run = 0.0f;
  const float sl2 = p.scale_log2;

  constexpr int STEP = PF_KEYS * PF_WAVES;
  // keys whose pages the table holds, wherever in a page they begin
  const int k_span = (int)min((int64_t)(PF_TABLE - 1) << shift, (int64_t)1 << 30) / STEP * STEP;
  for (int k_first = k_begin; k_first < k_end; k_first = k_stop) {
    if (k_first > k_begin) {
      wait_vmcnt<0>();
      __syncthreads();  // everyone is done with the table
    }
    k_stop = k_first + min(k_span, k_end - k_first);
    first_page = k_first >> shift;
    const int n_pages = ((k_stop - 1) >> shift) - first_page + 1;
    for (int i = threadIdx.x; i < n_pages; i += 64 * PF_WAVES)
      lds.table[i] = p.pv.pages[(int64_t)t.s * p.pv.pages_ld + first_page + i];
    __syncthreads();
    const int n_blocks = uniform((k_stop - k_first + PF_KEYS - 1) / PF_KEYS);
    int base = k_first + PF_KEYS * wave;
    uint32_t seen_now = 0, seen_next = 0;
    int stage = 0;
    if (wave >= n_blocks) continue;
    fetch(base, 0);
    seen_now = seen;
    fetch_k();
    fetch(base + STEP, 1);
    seen_next = seen;
    // Q is waited for here, or the loop's first product would wait for all that is on its way
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(qf[s]));
    for (int j = wave; j < n_blocks; j += PF_WAVES, base += STEP, stage ^= 1) {
      wait_vmcnt<NU>();  // only V of the next block, the last NU loads, may still be on its way
      asm volatile("" ::: "memory");
      const uint32_t st = ring + (uint32_t)(stage * L::BYTES);
      f32x4_t sc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[s][i]),
                                                         __builtin_bit_cast(bf16x8_t, qf[s]), sc[i], 0, 0, 0);
      fetch_k();  // of the next block
      // sc[t][e] is key 8g + 4t + e of row l16
      if (base + PF_KEYS > lim_lo || seen_now != ~0u) {
        const int room = lim - base;
        const uint32_t bits = (room >= 32 ? seen_now : room <= 0 ? 0u : seen_now & ((1u << room) - 1)) >> (8 * g);
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[i >> 2][i & 3] = (bits >> i) & 1 ? sc[i >> 2][i & 3] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sc[i >> 2][i & 3]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_old = m_run;
      const bool fresh = m_old == -INFINITY, raise = !fresh && (mx - m_old) * sl2 > PA_TAU;
      const float m_ref = fresh || raise ? mx : m_old;
      if (__any(raise)) {
        const float alpha = raise ? __builtin_amdgcn_exp2f((m_old - m_ref) * sl2) : 1.0f;
        l_run *= alpha;
#pragma unroll
        for (int c = 0; c < ND; ++c) o[c] *= alpha;
      }
      m_run = m_ref;
      const float nmc = m_ref == -INFINITY ? 0.0f : -m_ref * sl2;
      u32x4_t hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 1][2 * (i & 1)], sl2, nmc));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 1][2 * (i & 1) + 1], sl2, nmc));
        l_run += e0 + e1;
        hi[i] = pack_bf16x2(e0, e1);
        lo[i] = pack_bf16x2(e0 - bf16_bits_to_f32(hi[i] & 0xffffu), e1 - __uint_as_float(hi[i] & 0xffff0000u));
      }
      u32x4_t vf[ND];
      read_v<ND, 0, L::ROW>(vf, st, v_rd);
      __builtin_amdgcn_sched_barrier(0);  // nothing that the next block asks for comes before
      // V has been read: its place takes the block after next
      fetch(base + 2 * STEP, stage);
      seen_now = seen_next;
      seen_next = seen;
#pragma unroll
      for (int c = 0; c < ND; ++c) {
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                      __builtin_bit_cast(bf16x8_t, lo), o[c], 0, 0, 0);
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                      __builtin_bit_cast(bf16x8_t, hi), o[c], 0, 0, 0);
      }
    }
  }
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);

  // Join the waves: o[c][e] is component 16c + 4g + e of row l16.
  constexpr int PITCH = D + 4;  // floats, so that the rows' 16-byte stores spread over the banks
  static_assert(PF_ROWS * PITCH * 4 <= 2 * L::BYTES, "a wave's sums fit its ring");
  wait_vmcnt<0>();  // nothing is on its way to the ring any more
  __syncthreads();
  float* sums = (float*)(lds.ring + wave * 2 * L::BYTES);
#pragma unroll
  for (int c = 0; c < ND; ++c) *(f32x4_t*)(sums + l16 * PITCH + 16 * c + 4 * g) = o[c];
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
        s += f[w] * *(const f32x4_t*)((const float*)(lds.ring + w * 2 * L::BYTES) + r * PITCH + c);
      if (c >= p.d) continue;
      s *= inv;
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

template <int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) paged_attn_kernel(AttnParams p) {
  using L = PaLds<D>;
  constexpr int NS = D / 16, NC = D / 32, STAGE = 2 * L::BYTES;
  __shared__ union {
    __attribute__((aligned(16))) char ring[2 * STAGE];
    PfShared<D> few;
  } lds;
  const uint32_t lds0 = lds_addr(lds.ring);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int h32 = lane >> 5, l32 = lane & 31;

  // Workgroup b runs on XCD b mod 8.  With the KV heads innermost an XCD's L2 holds the keys of few of
  // them, which the row tiles of a sequence read at about the same time; the last tiles, which see the
  // most keys, come first.
  const int rest = uniform(blockIdx.x / p.n_kv), kvh = uniform(blockIdx.x - rest * p.n_kv);
  const int piece = uniform(rest / p.tiles), x = uniform(p.tiles - 1 - (rest - piece * p.tiles));
  const PaTile t = pa_tile(p, x);
  if (t.s < 0) return;
  const int end = t.end(p), plen = pa_piece(p, end);
  if (piece > 0 && (int64_t)piece * plen >= end) return;
  const int k_begin = piece * plen, k_end = k_begin + min(plen, end - k_begin);
  const bool whole = plen >= end;

  // this lane's row; rows past the sequence's last one repeat it and are not stored
  const int n_packed = min(t.n * p.group - t.first, PA_ROWS);
  // Decode rows beside prompts, and the ends of those: all four waves at one row tile (chunks of 500 and 63 rows over
  // 4000 keys: 44.9 us, 47.9 without; one of 500 and 63 single rows: 132.8, 129.8; 30 of up to 97 rows, 12 heads of
  // 64: 52.4, 53.0).
  if (n_packed <= PF_ROWS) {
    pf_segment<D>(p, lds.few, t, kvh, k_begin, k_end, whole,
                  [&](int row, int head) { return ((int64_t)piece * p.pv.total_q + row) * p.n_heads + head; });
    return;
  }
  const bool wave_has_rows = 32 * wave < n_packed;
  const int pr = t.first + min(32 * wave + l32, n_packed - 1);
  const int token = pr / p.group, head = kvh * p.group + pr - token * p.group;
  const int lim = t.limit(p, token);
  // the wave's rows see at least lim_lo and at most lim_hi keys
  const int lim_lo = t.limit(p, (t.first + min(32 * wave, n_packed - 1)) / p.group);
  const int lim_hi = t.limit(p, (t.first + min(32 * wave + 31, n_packed - 1)) / p.group);

  u32x4_t qf[NS];
  {
    const uint16_t* qr = p.q + (int64_t)(t.q0 + token) * p.q_t + (int64_t)head * p.q_h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = 8 * (2 * s + h32);
      qf[s] = c < p.d ? *(const u32x4_t*)(qr + c) : u32x4_t{0, 0, 0, 0};
    }
  }

  // DMA: wave w brings rows 16w .. 16w+15 of a block; in load u lane l brings a chunk of row
  // 16w + RPB*u + l/NCH.
  const uint16_t* kbase = p.k + (int64_t)kvh * p.pv.head_stride;
  const uint16_t* vbase = p.v + (int64_t)kvh * p.pv.head_stride;
  int page_next = -1;   // page of key `lane` of the next block to be issued, read a block ahead of its use
  uint64_t seen_next = 0;  // keys of the block issued last that exist
  auto look_up = [&](int base) __attribute__((always_inline)) {
    const int pos = base + lane;
    page_next = pos < k_end ? p.pv.pages[(int64_t)t.s * p.pv.pages_ld + (pos >> p.pv.page_shift)] : -1;
  };
  // The wave's 16 rows lie in one page where pages are of 16 tokens or more: a scalar base and these offsets.
  const bool even = p.pv.page_shift >= 4 && p.d == D && p.pv.slot_stride <= (1 << 24);
  uint32_t k_off[L::NU], v_off[L::NU];
#pragma unroll
  for (int u = 0; u < L::NU; ++u) {
    const int r = 16 * wave + L::RPB * u + lane / L::NCH, at = lane % L::NCH;
    k_off[u] = (uint32_t)((r & 15) * p.pv.slot_stride + 8 * L::k_pos(r, at));
    v_off[u] = (uint32_t)((r & 15) * p.pv.slot_stride + 8 * L::v_pos(r, at));
  }
  auto to_lds = [&](const uint16_t* src, uint32_t dst) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(uintptr_t)src,
                                     (__attribute__((address_space(3))) void*)(uintptr_t)dst, 16, 0, 0);
  };
  // asks for the block at `base`, whose pages have been looked up
  auto issue = [&](int base, int stage) __attribute__((always_inline)) {
    const bool there = (uint32_t)page_next < (uint32_t)p.pv.num_pages;
    const int mask = (1 << p.pv.page_shift) - 1;
    const uint32_t dst = lds0 + (uint32_t)(stage * STAGE + wave * L::NU * 1024);
    seen_next = __ballot(there);
    if (even && seen_next == ~uint64_t{0}) {
      const int64_t at = __builtin_amdgcn_readlane(page_next, 16 * wave) * p.pv.page_stride +
                         ((base + 16 * wave) & mask) * p.pv.slot_stride;
#pragma unroll
      for (int u = 0; u < L::NU; ++u) {
        to_lds(kbase + at + k_off[u], dst + u * 1024);
        to_lds(vbase + at + v_off[u], dst + u * 1024 + L::BYTES);
      }
      return;
    }
    const int64_t row_off = there ? page_next * p.pv.page_stride + ((base + lane) & mask) * p.pv.slot_stride : -1;
#pragma unroll
    for (int u = 0; u < L::NU; ++u) {
      const int r = 16 * wave + L::RPB * u + lane / L::NCH, at = lane % L::NCH;
      const int64_t off = __shfl(row_off, r, 64);
      const int kc = 8 * L::k_pos(r, at), vc = 8 * L::v_pos(r, at);
      to_lds(off >= 0 && kc < p.d ? kbase + off + kc : (const uint16_t*)pa_zero, dst + u * 1024);
      to_lds(off >= 0 && vc < p.d ? vbase + off + vc : (const uint16_t*)pa_zero, dst + u * 1024 + L::BYTES);
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

  // One 64-key block; `seen`: the keys that this lane's row sees, of which none is missing in any row of the
  // wave unless `masked`.
  auto block = [&](uint32_t st, uint64_t seen, bool masked) __attribute__((always_inline)) {
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
    static_for<4>([&](auto ks_c) __attribute__((always_inline)) {
      constexpr int ks = decltype(ks_c)::value;
      u32x4_t vf[NC];
      u32x4_t lo;
      {
        constexpr int kb = ks >> 1, base = 8 * (ks & 1);
#pragma unroll
        for (int w2 = 0; w2 < 4; ++w2)
          lo[w2] = pack_bf16x2(sc[kb][base + 2 * w2] - bf16_bits_to_f32(hi[ks][w2] & 0xffffu),
                               sc[kb][base + 2 * w2 + 1] - __uint_as_float(hi[ks][w2] & 0xffff0000u));
      }
      read_v<NC, 16 * ks * L::ROW, L::ROW>(vf, st, v_rd);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                       __builtin_bit_cast(bf16x8_t, lo), o[c], 0, 0, 0);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[c]),
                                                       __builtin_bit_cast(bf16x8_t, hi[ks]), o[c], 0, 0, 0);
    });
  };

  const int n_blocks = uniform((k_end - k_begin + PA_KEYS - 1) / PA_KEYS);
  if (n_blocks > 0) {
    look_up(k_begin);
    issue(k_begin, 0);
    look_up(k_begin + PA_KEYS);
  }
  for (int j = 0; j < n_blocks; ++j) {
    const uint64_t seen = seen_next;
    const int base = k_begin + j * PA_KEYS;
    wait_vmcnt<0>();     // this wave's share of block j has landed, and the pages of block j + 1
    lds_ring_barrier();  // and everyone's; and block j - 1 has been read
    if (j + 1 < n_blocks) {
      issue(base + PA_KEYS, (j + 1) & 1);
      look_up(base + 2 * PA_KEYS);
    }
    const uint32_t st = lds0 + (uint32_t)((j & 1) * STAGE);
    if (!wave_has_rows || base >= lim_hi) continue;
    const bool masked = base + PA_KEYS > lim_lo || seen != ~uint64_t{0};
    const int room = lim - base;
    block(st, room >= 64 ? seen : room <= 0 ? 0 : seen & ((uint64_t{1} << room) - 1), masked);
  }

  if (!wave_has_rows || 32 * wave + l32 >= n_packed) return;
  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
  const int64_t row = t.q0 + token;
  const float lse2 = l_tot == 0.0f ? -INFINITY : m_run * sl2 + __log2f(l_tot);
  if (whole) {
    uint16_t* out = p.o + row * p.o_t + (int64_t)head * p.o_h;
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

// A tile's keys in pieces, each a workgroup's.
template <int D>
__global__ void __launch_bounds__(64 * PF_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
    paged_attn_few_kernel(AttnParams p) {
  __shared__ PfShared<D> lds;
  // Workgroup b runs on XCD b mod 8: the heads and pieces of a tile go round all of them, so that a long
  // sequence does not keep one XCD busy alone, and begin one piece further on with each tile, so that the
  // first pieces, which every sequence has, do so too.
  const int inner = p.n_kv * p.pieces, x = uniform(blockIdx.x / inner);
  const int at_inner = uniform((int)((blockIdx.x % inner + (uint32_t)x % p.pieces * p.n_kv) % inner));
  const int kvh = uniform(at_inner % p.n_kv), piece = uniform(at_inner / p.n_kv);
  const PaTile t = pa_tile(p, x);
  if (t.s < 0) return;
  const int end = t.end(p), plen = pa_piece(p, end);
  if (piece > 0 && (int64_t)piece * plen >= end) return;
  const int k_begin = piece * plen;
  pf_segment<D>(p, lds, t, kvh, k_begin, k_begin + min(plen, end - k_begin), plen >= end,
                [&](int row, int head) { return ((int64_t)piece * p.pv.total_q + row) * p.n_heads + head; });
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

template <int D>
__global__ void __launch_bounds__(64 * PF_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
    paged_attn_share_kernel(AttnParams p) {
  __shared__ PfShared<D> lds;
  __shared__ uint32_t prefix[PF_SEQS + 1], wave_sum[PF_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, S = p.pv.n_seqs;
  const int kvh = uniform(blockIdx.x % p.n_kv);
  const uint32_t w = uniform((int)(blockIdx.x / p.n_kv));
  constexpr int EACH = PF_SEQS / (64 * PF_WAVES);
  uint32_t n[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = EACH * tid + i;
    n[i] = s < S ? (uint32_t)(min(max(p.pv.kv_len[s], 0), p.cap) + PF_BLOCK - 1) / PF_BLOCK : 0;
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
    const int k_begin = (int)(b - first) * PF_BLOCK, k_end = last == next ? len : (int)(last - first) * PF_BLOCK;
    pf_segment<D>(p, lds, t, kvh, k_begin, k_end, b == first && last == next,
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

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

size_t mi_paged_attn_workspace_size(int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t n_seqs, int64_t total_q,
                                    int64_t max_q_len, int64_t max_kv_len) {
  if (n_heads < 1 || n_kv < 1 || n_heads % n_kv || head_dim < 1 || n_seqs < 1 || total_q < 1) return 0;
  if (n_seqs > INT32_MAX || total_q > INT32_MAX / n_heads) return 0;  // refused by the call
  // CUs of the current device, whose table the first of all calls fills in; without one, those of an MI355X
  const int cus = host_device() == MI_OK ? host_cus() : 256;
  const PaPlan plan = pa_plan(n_heads, n_kv, head_dim, n_seqs, total_q, max_q_len, max_kv_len,
                              total_q == n_seqs && max_q_len == 1, cus);
  return (size_t)std::max(plan.bytes(total_q, n_heads, head_dim), plan.share_bytes(n_seqs, n_heads, head_dim));
}

int mi_paged_attn(void* stream, const void* Q, int64_t q_t, int64_t q_h, void* O, int64_t o_t, int64_t o_h, float* lse,
                  int64_t n_heads, const mi_paged_cache* cache, const mi_paged_seqs* seqs, int64_t max_q_len,
                  int64_t max_kv_len, int32_t causal, float scale, void* workspace, size_t workspace_bytes) {
  int st = check_paged(cache, seqs);
  if (st != MI_OK) return st;
  if (n_heads < 0 || max_q_len < 0 || max_kv_len < 0) return host_fail(MI_ERR_SHAPE, "negative size");
  if (seqs->n_seqs == 0 || seqs->total_q == 0 || n_heads == 0) return MI_OK;
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
  if (!(scale > 0.0f) || !isfinite(scale * 1.4426950408889634f)) return host_fail(MI_ERR_UNSUPPORTED, "scale must be positive and finite");
  if (rows * n_heads > INT32_MAX) return host_fail(MI_ERR_SHAPE, "total_q * n_heads exceeds 2^31-1");
  st = host_device();
  if (st != MI_OK) return st;
  PaPlan plan = pa_plan(n_heads, cache->n_kv, d, seqs->n_seqs, rows, max_q_len, max_kv_len, !seqs->q_start, host_cus());
  if (seqs->n_seqs * (seqs->max_pages * cache->page_size / PF_BLOCK + 1) > INT32_MAX) plan.share = 0;  // its sums
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
  p.tile_shift = plan.tile_shift;
  p.tiles = (int)plan.tiles;
  p.pieces = plan.pieces;
  p.min_piece = plan.min_piece;
  p.cap = (int)(seqs->max_pages * cache->page_size);
  p.part_o = (float*)workspace;
  p.part_lse = p.part_o ? p.part_o + plan.pieces * rows * n_heads * d : nullptr;
  p.share = 0;
  p.prefix = nullptr;
  p.scale_log2 = scale * 1.4426950408889634f;
  hipError_t e;
  if (plan.share && workspace && plan.share_bytes(rows, n_heads, d) <= (int64_t)workspace_bytes) {
    p.share = plan.share;
    p.part_lse = p.part_o + 2 * (int64_t)p.share * n_heads * d;
    p.prefix = (uint32_t*)(p.part_lse + 2 * (int64_t)p.share * n_heads);
    const unsigned wgs = (unsigned)(p.share * p.n_kv);
    if (d <= 64) paged_attn_share_kernel<64><<<wgs, 64 * PF_WAVES, 0, (hipStream_t)stream>>>(p);
    else paged_attn_share_kernel<128><<<wgs, 64 * PF_WAVES, 0, (hipStream_t)stream>>>(p);
    e = hipGetLastError();
    if (e == hipSuccess) {
      paged_attn_share_join_kernel<<<(unsigned)(rows * n_heads), 256, 0, (hipStream_t)stream>>>(p);
      e = hipGetLastError();
    }
    return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "paged_attn launch: %s", hipGetErrorString(e));
  }
  const int64_t grid = plan.tiles * p.n_kv * plan.pieces, most = host_most_groups(256);
  if (grid > most)
    return host_fail(MI_ERR_SHAPE, "%lld row tiles of %lld KV heads: more than %lld workgroups", (long long)plan.tiles,
                     (long long)cache->n_kv, (long long)most);
  if (plan.few) {
    if (d <= 64) paged_attn_few_kernel<64><<<(unsigned)grid, 64 * PF_WAVES, 0, (hipStream_t)stream>>>(p);
    else paged_attn_few_kernel<128><<<(unsigned)grid, 64 * PF_WAVES, 0, (hipStream_t)stream>>>(p);
  } else if (d <= 64) paged_attn_kernel<64><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(p);
  else paged_attn_kernel<128><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(p);
  e = hipGetLastError();
  if (e == hipSuccess && plan.pieces > 1) {
    const unsigned wgs8 = (unsigned)(rows * ((n_heads + 7) / 8));
    if (plan.pieces <= 8 && !plan.few) paged_attn_join8_kernel<<<wgs8, 256, 0, (hipStream_t)stream>>>(p);
    else paged_attn_join_kernel<<<(unsigned)(rows * n_heads), 256, 0, (hipStream_t)stream>>>(p);
    e = hipGetLastError();
  }
  return e == hipSuccess ? MI_OK : host_fail(MI_ERR_HIP, "paged_attn launch: %s", hipGetErrorString(e));
}

}  // extern "C"
