// mi_paged.hip -- attention of a chunk of new tokens over a paged K/V cache in bf16, gfx950.
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
#include "mi_paged_attn.hpp"

namespace mig {
namespace {

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
struct PfShared {
  __attribute__((aligned(16))) char ring[PF_WAVES * 2 * PfLds<D>::BYTES];
  int table[PF_TABLE];
  PfWaves waves;
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

  const uint16_t* kbase = (const uint16_t*)p.k + (int64_t)kvh * p.pv.head_stride;
  const uint16_t* vbase = (const uint16_t*)p.v + (int64_t)kvh * p.pv.head_stride;
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
      read_v<ND, 0, 4 * L::ROW>(vf, st, v_rd);
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
  static_assert(PF_ROWS * PF_PITCH<D> * 4 <= 2 * L::BYTES, "a wave's sums fit its ring");
  wait_vmcnt<0>();  // nothing is on its way to the ring any more
  pf_join_waves<D>(p, lds.ring, 2 * L::BYTES, lds.waves, t, kvh, n_packed, o, m_run, l_run, whole, part_at,
                   [](int, int) { return 0u; });
}

template <int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) paged_attn_kernel(AttnParams p) {
  using L = PaLds<D>;
  constexpr int STAGE = 2 * L::BYTES;
  __shared__ union {
    __attribute__((aligned(16))) char ring[2 * STAGE];
    PfShared<D> few;
  } lds;
  const uint32_t lds0 = lds_addr(lds.ring);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);

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
  PaRows<D, true> rows;
  rows.begin(p, t, kvh, wave, n_packed);

  // DMA: wave w brings rows 16w .. 16w+15 of a block; in load u lane l brings a chunk of row
  // 16w + RPB*u + l/NCH.
  const uint16_t* kbase = (const uint16_t*)p.k + (int64_t)kvh * p.pv.head_stride;
  const uint16_t* vbase = (const uint16_t*)p.v + (int64_t)kvh * p.pv.head_stride;
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
    if (wave_has_rows) rows.block(st, base, seen);
  }
  if (wave_has_rows) rows.end(p, t, wave, n_packed, piece, whole, [](int) { return 0u; });
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

template <int D>
__global__ void __launch_bounds__(64 * PF_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
    paged_attn_share_kernel(AttnParams p) {
  __shared__ PfShared<D> lds;
  __shared__ PfPrefix prefix;
  const int kvh = uniform(blockIdx.x % p.n_kv);
  pf_over_share<0>(p, prefix, uniform((int)(blockIdx.x / p.n_kv)),
                   [&](const PaTile& t, int k_begin, int k_end, bool whole, auto part_at) __attribute__((always_inline)) {
                     pf_segment<D>(p, lds, t, kvh, k_begin, k_end, whole, part_at);
                   });
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

size_t mi_paged_attn_workspace_size(int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t n_seqs, int64_t total_q,
                                    int64_t max_q_len, int64_t max_kv_len) {
  return pa_workspace_size(n_heads, n_kv, head_dim, n_seqs, total_q, max_q_len, max_kv_len);
}

int mi_paged_attn(void* stream, const void* Q, int64_t q_t, int64_t q_h, void* O, int64_t o_t, int64_t o_h, float* lse,
                  int64_t n_heads, const mi_paged_cache* cache, const mi_paged_seqs* seqs, int64_t max_q_len,
                  int64_t max_kv_len, int32_t causal, float scale, void* workspace, size_t workspace_bytes) {
  int st = check_paged(cache, seqs);
  if (st != MI_OK) return st;
  AttnParams p;
  PaPlan plan;
  bool launch;
  st = pa_prepare(p, plan, launch, Q, q_t, q_h, O, o_t, o_h, lse, n_heads, cache->n_kv, cache->head_dim, cache->page_size,
                  seqs, paged_view(cache, seqs), max_q_len, max_kv_len, causal, scale, workspace, workspace_bytes);
  if (st != MI_OK || !launch) return st;
  p.k = cache->k;
  p.v = cache->v;
  hipStream_t hs = (hipStream_t)stream;
  const bool small = cache->head_dim <= 64;
  return pa_launch(
      p, plan, hs,
      [&](unsigned wgs) {
        if (small) paged_attn_share_kernel<64><<<wgs, 64 * PF_WAVES, 0, hs>>>(p);
        else paged_attn_share_kernel<128><<<wgs, 64 * PF_WAVES, 0, hs>>>(p);
      },
      [&](unsigned wgs) {
        if (small) paged_attn_few_kernel<64><<<wgs, 64 * PF_WAVES, 0, hs>>>(p);
        else paged_attn_few_kernel<128><<<wgs, 64 * PF_WAVES, 0, hs>>>(p);
      },
      [&](unsigned wgs) {
        if (small) paged_attn_kernel<64><<<wgs, 256, 0, hs>>>(p);
        else paged_attn_kernel<128><<<wgs, 256, 0, hs>>>(p);
      });
}

}  // extern "C"
