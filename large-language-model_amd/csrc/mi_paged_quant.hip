// mi_paged_quant.hip -- attention of new tokens over a paged K/V cache of 8 or 4 bits, gfx950.
//
// The formula, the tiles, pieces, shares and joins are those of the cache in bf16 (mi_paged.hip, mi_paged_attn.hpp);
// here the keys and values come as codes and a power of two for 32 of them.  The conversion gives two bf16 at once
// and multiplies on the way, both exactly, so scores and sums are those of a bf16 cache that holds the values
// which the codes stand for.
//
// A quarter of a row of up to D = 64 or 128 components is what a lane loads and converts: D / 4 of them, within one
// group.  Quarters past head_dim are zeros that are multiplied like the others: half of them in heads of 32, one of
// four in heads of 96.
//
// Few rows are bound by HBM where the keys are many, else by a wave's chain for a block (0.6 us with one wave a SIMD);
// many by their waves' chains of products and exponentials: a 64-key block of 128 rows takes 1.6 us alone in a CU, 2.3
// beside a second workgroup and 4.2 beside two (heads of 64; of 128 in 4 bits 2.4 and 4.8), and with all pages in the
// caches at most 4 % less, so its loads, one block ahead, are not what it waits for.  On an MI355X: 64 x 32768 keys at 5.2 TB/s
// in 4 bits (with no arithmetic at all 5.5) and 5.7 to 5.9 in 8 bits; 64 sequences of 500 to 8000 keys in 4 bits 28.1
// us (in bf16 77.5), 16 in 8 bits 39 (70); four chunks of 1024 rows over 4095 keys 75 (69.5), of whose busy CUs' clocks
// the matrix cores have 44 % and vector instructions 56 %.
//
// The plan's borders are those of the cache in bf16 (pa_plan), and hold here (us, 16 / 4 heads of 128, 4 bits). One piece
// / pieces of 128 keys: 512 keys 8.5 / 9.7, 1024 keys 11.5 / 9.8.  Pieces / even shares, which the
// last two columns take:
//    sequences x keys   64 x 2000   256 x 2000   16 x 4000    16 x 8000    64 x 8000
//              uneven   19.2/17.0   31.7/36.1    15.1/13.9    22.2/15.7    55.4/28.4
//                even   20.3/22.9   50.2/54.4    16.5/16.4    23.3/22.8    57.7/51.7
// Many rows: twice as many pieces or longer ones took the chunks to 72 at best, mixed rows from 34.4 to 34.5.
#include <hip/hip_runtime.h>

#include "mi_kv_quant.hpp"
#include "mi_paged_attn.hpp"

namespace mig {
namespace {

struct QuantParams : AttnParams {
  const uint8_t *ks, *vs;
  int64_t scale_page, scale_head, scale_slot;
};

// A quarter of a row of up to D components: its codes, and how they become bf16.
template <int D, int BITS>
struct Quarter {
  static constexpr int COMPS = D / 4, BYTES = COMPS * BITS / 8, EIGHTS = COMPS / 8;
  uint32_t w[BYTES / 4];
  uint32_t scale;  // the byte
  // by global loads whatever the compiler knows of the addresses: flat ones would count as LDS accesses, too
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales) {
#define MIG_GLOBAL(T, p) ((const __attribute__((address_space(1))) T*)(uintptr_t)(p))
    if constexpr (BYTES == 8) *(u32x2_t*)w = *MIG_GLOBAL(u32x2_t, codes);
    else
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) ((u32x4_t*)w)[i] = MIG_GLOBAL(u32x4_t, codes)[i];
    scale = *MIG_GLOBAL(uint8_t, scales);
#undef MIG_GLOBAL
  }
  __device__ __forceinline__ u32x4_t eight(int i) const { return kv_eight<BITS>(w + i * (BITS / 4), kv_power(scale)); }
  // Eighths i and i ^ bit in each other's place, if `is`.
  __device__ __forceinline__ void swap(int bit, bool is) {
    constexpr int N = BITS / 4;  // dwords of an eighth
#pragma unroll
    for (int i = 0; i < EIGHTS; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (!(i & bit) && (i | bit) < EIGHTS) {
          const uint32_t a = w[i * N + n], b = w[(i | bit) * N + n];
          w[i * N + n] = is ? b : a;
          w[(i | bit) * N + n] = is ? a : b;
        }
  }
  // e4m3's codes of NaN, 0x7f and 0xff, in dword i: bit 7 of their bytes.
  __device__ __forceinline__ uint32_t nan_codes(int i) const { return ((w[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
  // Whether component c of the quarter reads back as NaN.
  __device__ __forceinline__ bool nan(int c) const {
    return scale == 255 || (BITS == 8 && (nan_codes(c / 4) >> (8 * (c & 3) + 7)) & 1);
  }
  // What reads back as NaN becomes zero, or under byte 0 at least finite, if it had byte 255; whether there was any.
  __device__ __forceinline__ bool hide() {
    bool any = scale == 255;
    scale = any ? 0 : scale;
    if constexpr (BITS == 8) {
      uint32_t codes = 0;
#pragma unroll
      for (int i = 0; i < BYTES / 4; ++i) codes |= nan_codes(i);
      if (codes) {
        any = true;
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) {
          const uint32_t m = nan_codes(i);
          w[i] &= ~(m | (m - (m >> 7)));
        }
      }
    }
    return any;
  }
};

// NaN of V among keys that not every row of a tile sees.  A weight of 0 times NaN is NaN, so there it is held as zeros;
// where any was, the workgroup looks at the keys [from, to) once more at the end for the first one at which each component
// is NaN, and the rows that see it get their NaN.  The append writes NaN by whole groups; a cache that something else
// has filled may hold codes of NaN, too.
template <int D, int BITS>
struct PqNan {
  using Q4 = Quarter<D, BITS>;
  const int* first;  // [D] in LDS
  bool any = false;
  __device__ __forceinline__ PqNan(const int* table) : first(table) {}
  // All threads together; table: D entries of LDS that nothing reads any more once everyone has come here.
  __device__ __forceinline__ void look(const QuantParams& p, const PaTile& t, int kvh, int from, int to, int* table) {
    any = true;
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += blockDim.x) table[i] = INT32_MAX;
    __syncthreads();
    const int quarter = threadIdx.x & 3, c0 = Q4::COMPS * quarter;
    for (int key = from + (int)(threadIdx.x >> 2); key < to; key += blockDim.x >> 2) {
      const int page = page_of(p.pv, t.s, key), slot = key & ((1 << p.pv.page_shift) - 1);
      if (page < 0 || c0 >= p.d) continue;
      Q4 v;
      v.load((const uint8_t*)p.v + kvh * p.pv.head_stride + page * p.pv.page_stride + slot * p.pv.slot_stride +
                 Q4::BYTES * quarter,
             p.vs + kvh * p.scale_head + page * p.scale_page + slot * p.scale_slot + c0 / KV_GROUP);
      for (int c = 0; c < Q4::COMPS; ++c)
        if (v.nan(c)) atomicMin(&table[c0 + c], key);
    }
    __syncthreads();
  }
  // bit i: a row of `lim` keys sees a NaN of component 32c + i
  __device__ __forceinline__ uint32_t seen(int lim, int c) const {
    uint32_t comps = 0;
    if (any)
      for (int i = 0; i < 32; ++i) comps |= lim > first[32 * c + i] ? 1u << i : 0;
    return comps;
  }
};

// Codes and scale bytes of keys that no row sees, and of components past head_dim: zeros under byte 0, which are zeros.
__device__ __align__(16) uint32_t pq_zero[8];

// Few rows: V of a 32-key block of a wave, converted, rows of D components whose 16-byte chunks are moved so that
// nothing collides: a write's lanes have 128 bytes a clock, the quarters of two rows (32 banks), a transposing
// read's 256, 32 bytes of each of eight rows (64 banks).  Rows 8 apart have one order.
template <int D>
struct PqLds {
  static constexpr int ROW = D * 2;
  static constexpr int V_BYTES = PF_KEYS * ROW;
  static constexpr int SUM_BYTES = PF_ROWS * PF_PITCH<D> * 4;
  static constexpr int BYTES = V_BYTES > SUM_BYTES ? V_BYTES : SUM_BYTES;
  __device__ static __forceinline__ int v_pos(int r, int c) {
    if constexpr (D == 128) return c ^ ((r & 7) << 1) ^ (c >> 3);
    else return c ^ (r & 7);
  }
};

template <int D>
struct PqShared {
  __attribute__((aligned(16))) char v[PF_WAVES * PqLds<D>::BYTES];
  int table[PF_TABLE];
  PfWaves waves;
  int hidden[PF_WAVES];  // of each: whether it held a NaN as zero
};

// Keys [k_begin, k_end) of a tile of KV head kvh; whole: they are all its keys, and O and lse are written; else the
// part, at part_at(row of the sequence, head).  Every wave takes 32-key blocks of its own, whose codes come into
// registers DEPTH blocks ahead: with one more the steady rate is the same, and a segment starts and ends later (64
// sequences of 500 to 8000 keys in 4 bits 28.5 us, so 29.9 beside it; 16 in 8 bits 38.6 and 39.9).  One load for all scale
// bytes of a block, given to the lanes by shuffles, was slower (30.6): it makes the chain longer.
// ONE: the tile's rows are of one token.
template <int D, int BITS, bool ONE, class PartAt>
__device__ __forceinline__ void pq_segment(const QuantParams& p, PqShared<D>& lds, const PaTile& t, int kvh, int k_begin,
                                           int k_end, bool whole, PartAt part_at) {
  using L = PqLds<D>;
  using Q4 = Quarter<D, BITS>;
  constexpr int NS = D / 32, ND = D / 16, DEPTH = 2, STEP = PF_KEYS * PF_WAVES;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // or what a segment needs at its ends would be kept in registers from one to the next
  const int wave = uniform(threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
  const uint32_t vlds = lds_addr(lds.v) + (uint32_t)(wave * L::BYTES);

  const int n_packed = min(t.n * p.group - t.first, PF_ROWS);
  const int pr = t.first + min(l16, n_packed - 1);
  const int token = pr / p.group, head = kvh * p.group + pr - token * p.group;
  const int lim = t.limit(p, token), lim_lo = t.limit(p, t.first / p.group);
  const bool uneven = !ONE && lim_lo < t.end(p);
  if (!ONE) lds.hidden[wave] = 0;

  // lane (g, l16) holds the components of quarter g of K's row and of Q's: product s takes eight of each quarter
  u32x4_t qf[NS];
  {
    const uint16_t* qr = p.q + (int64_t)(t.q0 + token) * p.q_t + (int64_t)head * p.q_h;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = Q4::COMPS * g + 8 * s;
      qf[s] = c < p.d ? *(const u32x4_t*)(qr + c) : u32x4_t{0, 0, 0, 0};
    }
  }

  const int shift = p.pv.page_shift;
  const int64_t slot_stride = p.pv.slot_stride;
  const uint8_t* kbase = (const uint8_t*)p.k + kvh * p.pv.head_stride;
  const uint8_t* vbase = (const uint8_t*)p.v + kvh * p.pv.head_stride;
  const uint8_t* ksbase = p.ks + kvh * p.scale_head;
  const uint8_t* vsbase = p.vs + kvh * p.scale_head;
  int first_page = 0, k_stop = 0;  // the table holds the pages of the keys before k_stop

  // Tile i of the scores: row r reads key 16i + r, so the eight scores of a lane are the keys 4g + e and 16 + 4g + e,
  // e = 0 .. 3, and the second operand of P V takes these.  V: row 16u + lane / 4, quarter lane % 4.
  const int v_row = lane >> 2, v_q = lane & 3;
  const bool k_in = Q4::COMPS * g < p.d, v_in = Q4::COMPS * v_q < p.d;  // d is a multiple of 32: whole quarters
  const int k_code = Q4::BYTES * g, k_scale = Q4::COMPS * g / KV_GROUP;
  const int v_code = Q4::BYTES * v_q, v_scale = Q4::COMPS * v_q / KV_GROUP;
  // Whole blocks whose halves lie in one page each: scalar bases, of products of 32 bits each, and these offsets.
  const int64_t most32 = INT32_MAX;
  const bool even = shift >= 4 && p.d == D && p.pv.page_stride <= most32 && slot_stride << shift <= most32 &&
                    p.scale_page <= most32 && p.scale_slot << shift <= most32;
  const uint32_t page32 = (uint32_t)p.pv.page_stride, slot32 = (uint32_t)slot_stride;
  const uint32_t spage32 = (uint32_t)p.scale_page, sslot32 = (uint32_t)p.scale_slot;
  const uint32_t k_off = l16 * slot32 + k_code, ks_off = l16 * sslot32 + k_scale;
  const uint32_t v_off = v_row * slot32 + v_code, vs_off = v_row * sslot32 + v_scale;
  const int mask = (1 << shift) - 1;
  struct Block {
    Q4 k[2], v[2];
    uint32_t seen;  // its keys that exist
  } ring[DEPTH];
  int page_lo, page_hi;  // of the halves of the block to be asked for next, read a block ahead of their use
  auto look_up = [&](int base) __attribute__((always_inline)) {
    page_lo = lds.table[(min(base, k_stop - 1) >> shift) - first_page];
    page_hi = lds.table[(min(base + 16, k_stop - 1) >> shift) - first_page];
  };
  // Asks for the block at `base`, whose pages have been looked up.  A block past the end is asked for from zeros,
  // so that every step has the same loads on their way and waits for no more than its own.
  auto fetch = [&](Block& b, int base) __attribute__((always_inline)) {
    const uint32_t p0 = (uint32_t)uniform(page_lo), p1 = (uint32_t)uniform(page_hi);
    const uint8_t *kp[2], *ksp[2], *vp[2], *vsp[2];
    uint32_t seen = ~0u;
    if (even && base + PF_KEYS <= k_stop && p0 < (uint32_t)p.pv.num_pages && p1 < (uint32_t)p.pv.num_pages) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t page = i ? p1 : p0, slot = (base + 16 * i) & mask;
        const uint64_t at = (uint64_t)page * page32 + slot * slot32, sat = (uint64_t)page * spage32 + slot * sslot32;
        kp[i] = kbase + at + k_off, ksp[i] = ksbase + sat + ks_off;
        vp[i] = vbase + at + v_off, vsp[i] = vsbase + sat + vs_off;
      }
    } else if (base >= k_stop) {
      seen = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) kp[i] = ksp[i] = vp[i] = vsp[i] = (const uint8_t*)pq_zero;
    } else {
      const int pos = base + (lane & 31);
      const int page = lds.table[(min(pos, k_stop - 1) >> shift) - first_page];
      const bool there = pos < k_stop && (uint32_t)page < (uint32_t)p.pv.num_pages;
      const int slot = pos & mask;
      const int64_t off = there ? page * p.pv.page_stride + slot * slot_stride : -1;
      const int64_t soff = page * p.scale_page + slot * p.scale_slot;
      seen = (uint32_t)__ballot(there);
      const uint8_t* zero = (const uint8_t*)pq_zero;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t ko = __shfl(off, 16 * i + l16, 64), kso = __shfl(soff, 16 * i + l16, 64);
        const int64_t vo = __shfl(off, 16 * i + v_row, 64), vso = __shfl(soff, 16 * i + v_row, 64);
        const bool k_ok = ko >= 0 && k_in, v_ok = vo >= 0 && v_in;
        kp[i] = k_ok ? kbase + ko + k_code : zero, ksp[i] = k_ok ? ksbase + kso + k_scale : zero;
        vp[i] = v_ok ? vbase + vo + v_code : zero, vsp[i] = v_ok ? vsbase + vso + v_scale : zero;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      b.k[i].load(kp[i], ksp[i]);
      b.v[i].load(vp[i], vsp[i]);
    }
    b.seen = seen;
    look_up(base + STEP);
  };

  uint32_t v_rd[ND], v_wr[Q4::EIGHTS];
#pragma unroll
  for (int c = 0; c < ND; ++c) {
    const int r = 4 * g + (l16 >> 2), col = 16 * c + 4 * (l16 & 3);
    v_rd[c] = vlds + (uint32_t)(r * L::ROW + 16 * L::v_pos(r, col >> 3) + (col & 7) * 2);
  }
#pragma unroll
  for (int j = 0; j < Q4::EIGHTS; ++j)
    v_wr[j] = vlds + (uint32_t)(v_row * L::ROW + 16 * L::v_pos(v_row, Q4::EIGHTS * v_q + j));

  f32x4_t o[ND];
#pragma unroll
  for (int c = 0; c < ND; ++c) o[c] = f32x4_t{0, 0, 0, 0};
  // the row's reference maximum, what a score has to exceed to move it, and -m_run in log2 units
  float m_run = -INFINITY, l_run = 0.0f, m_lim = -INFINITY, nmc = 0.0f;
  const float sl2 = p.scale_log2, tau = PA_TAU / sl2;

  // V's fragment c, channels 16c + l16 by the keys that sc has, from where its block was written
  auto v_frag = [&](int c) __attribute__((always_inline)) {
    const u32x2_t lo = read_tr16(v_rd[c]), hi = read_tr16(v_rd[c] + 16 * L::ROW);
    return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
  };
  auto work = [&](Block& b, int base) __attribute__((always_inline)) {
    if (uneven && base + PF_KEYS > lim_lo) {
      if (b.v[0].hide()) lds.hidden[wave] = 1;
      if (b.v[1].hide()) lds.hidden[wave] = 1;
    }
    // V goes through LDS, which serves a wave in order, to its transposing reads
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < Q4::EIGHTS; ++j) *(lds_u32x4_t*)(uintptr_t)(v_wr[j] + u * 16 * L::ROW) = b.v[u].eight(j);
    f32x4_t sc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b.k[i].eight(s)),
                                                       __builtin_bit_cast(bf16x8_t, qf[s]), sc[i], 0, 0, 0);
    u32x4_t vf[ND / 2];
#pragma unroll
    for (int c = 0; c < ND / 2; ++c) vf[c] = v_frag(c);
    // sc[t][e] is key 16t + 4g + e of row l16
    if (base + PF_KEYS > lim_lo || b.seen != ~0u) {
      const int room = lim - base;
      const uint32_t bits = (room >= 32 ? b.seen : room <= 0 ? 0u : b.seen & ((1u << room) - 1)) >> (4 * g);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        sc[i >> 2][i & 3] = (bits >> (16 * (i >> 2) + (i & 3))) & 1 ? sc[i >> 2][i & 3] : -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sc[i >> 2][i & 3]);
    // Lanes l16 + 16g share a row and its reference maximum.  It is moved, and the lanes' maxima looked at
    // together, only where one of them has a first score or one that exceeds it by PA_TAU.
    if (__any(mx > m_lim)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const bool raise = mx > m_lim;
      const float m_ref = raise ? mx : m_run;
      const float alpha = raise && m_run != -INFINITY ? __builtin_amdgcn_exp2f((m_run - m_ref) * sl2) : 1.0f;
      l_run *= alpha;
#pragma unroll
      for (int c = 0; c < ND; ++c) o[c] *= alpha;
      m_run = m_ref;
      m_lim = m_run == -INFINITY ? -INFINITY : m_run + tau;
      nmc = m_run == -INFINITY ? 0.0f : -m_run * sl2;
    }
    u32x4_t hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 1][2 * (i & 1)], sl2, nmc));
      const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 1][2 * (i & 1) + 1], sl2, nmc));
      l_run += e0 + e1;
      hi[i] = pack_bf16x2(e0, e1);
      lo[i] = pack_bf16x2(e0 - bf16_bits_to_f32(hi[i] & 0xffffu), e1 - __uint_as_float(hi[i] & 0xffff0000u));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < ND / 2; ++i) {
        const int c = h * ND / 2 + i;
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[i]),
                                                      __builtin_bit_cast(bf16x8_t, lo), o[c], 0, 0, 0);
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf[i]),
                                                      __builtin_bit_cast(bf16x8_t, hi), o[c], 0, 0, 0);
        if (h == 0) vf[i] = v_frag(ND / 2 + i);
      }
  };

  // keys whose pages the table holds, wherever in a page they begin
  const int k_span = (int)min((int64_t)(PF_TABLE - 1) << shift, (int64_t)1 << 30) / STEP * STEP;
  for (int k_first = k_begin; k_first < k_end; k_first = k_stop) {
    if (k_first > k_begin) __syncthreads();  // everyone is done with the table
    k_stop = k_first + min(k_span, k_end - k_first);
    first_page = k_first >> shift;
    const int n_pages = ((k_stop - 1) >> shift) - first_page + 1;
    for (int i = threadIdx.x; i < n_pages; i += 64 * PF_WAVES)
      lds.table[i] = p.pv.pages[(int64_t)t.s * p.pv.pages_ld + first_page + i];
    __syncthreads();
    int base = k_first + PF_KEYS * wave;
    if (base >= k_stop) continue;
    look_up(base);
    static_for<DEPTH>([&](auto i) __attribute__((always_inline)) { fetch(ring[i], base + STEP * i); });
    auto step = [&](Block& b) __attribute__((always_inline)) {
      work(b, base);
      fetch(b, base + STEP * DEPTH);
      base += STEP;
      return base < k_stop;
    };
    static_assert(DEPTH == 2, "written out for two");
    while (step(ring[0]) && step(ring[1])) {
    }
  }
  PqNan<D, BITS> nan(lds.table);
  __syncthreads();  // V's place takes the waves' sums
  if (!ONE && (lds.hidden[0] | lds.hidden[1] | lds.hidden[2] | lds.hidden[3]))
    nan.look(p, t, kvh, max(k_begin, lim_lo - PF_KEYS + 1), k_end, lds.table);
  pf_join_waves<D>(p, lds.v, L::BYTES, lds.waves, t, kvh, n_packed, o, m_run, l_run, whole, part_at,
                   [&](int token, int c) { return ONE ? 0u : nan.seen(t.limit(p, token), c); });
}

// Many rows: a workgroup converts each 64-key block once, into LDS as the cache in bf16 would have it, and its waves
// multiply from there.
template <int D, int BITS>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) paged_attn_quant_kernel(QuantParams p) {
  using L = PaLds<D>;
  using Q4 = Quarter<D, BITS>;
  constexpr int STAGE = 2 * L::BYTES;
  __shared__ union {
    __attribute__((aligned(16))) char ring[2 * STAGE];
    PqShared<D> few;
  } lds;
  __shared__ int hidden[4];  // of each wave: whether it held a NaN as zero
  const uint32_t lds0 = lds_addr(lds.ring);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);

  // KV heads innermost, the last tiles, which see the most keys, first (as in mi_paged.hip)
  const int rest = uniform(blockIdx.x / p.n_kv), kvh = uniform(blockIdx.x - rest * p.n_kv);
  const int piece = uniform(rest / p.tiles), x = uniform(p.tiles - 1 - (rest - piece * p.tiles));
  const PaTile t = pa_tile(p, x);
  if (t.s < 0) return;
  const int end = t.end(p), plen = pa_piece(p, end);
  if (piece > 0 && (int64_t)piece * plen >= end) return;
  const int k_begin = piece * plen, k_end = k_begin + min(plen, end - k_begin);
  const bool whole = plen >= end;

  const int n_packed = min(t.n * p.group - t.first, PA_ROWS);
  if (n_packed <= PF_ROWS) {
    pq_segment<D, BITS, false>(p, lds.few, t, kvh, k_begin, k_end, whole,
                        [&](int row, int head) { return ((int64_t)piece * p.pv.total_q + row) * p.n_heads + head; });
    return;
  }
  const bool wave_has_rows = 32 * wave < n_packed;
  PaRows<D, false> rows;
  rows.begin(p, t, kvh, wave, n_packed);

  // wave w brings rows 16w .. 16w+15 of a block, a lane a quarter of row 16w + lane / 4
  const int row = 16 * wave + (lane >> 2), quarter = lane & 3;
  const bool in = Q4::COMPS * quarter < p.d;
  const int code_at = Q4::BYTES * quarter, scale_at = Q4::COMPS * quarter / KV_GROUP;
  const uint8_t* kbase = (const uint8_t*)p.k + kvh * p.pv.head_stride + code_at;
  const uint8_t* vbase = (const uint8_t*)p.v + kvh * p.pv.head_stride + code_at;
  const uint8_t* ksbase = p.ks + kvh * p.scale_head + scale_at;
  const uint8_t* vsbase = p.vs + kvh * p.scale_head + scale_at;
  // Eight lanes write at once, the quarters of two rows, whose eighths j lie in two or four of the eight places of 16 bytes:
  // so lanes write theirs in orders of their own, j ^ turn (four chunks of 1024 rows in 4 bits 76.7 us, so 75.0).
  const int k_turn = D == 128 ? quarter & 2 : row & 1;
  const int v_turn = D == 128 ? (row & 1) << 1 | quarter >> 1 : row & 1;
  uint32_t k_wr[Q4::EIGHTS], v_wr[Q4::EIGHTS];
#pragma unroll
  for (int j = 0; j < Q4::EIGHTS; ++j) {
    k_wr[j] = (uint32_t)(row * L::ROW + 16 * L::k_pos(row, Q4::EIGHTS * quarter + (j ^ k_turn)));
    v_wr[j] = (uint32_t)(L::BYTES + row * L::ROW + 16 * L::v_pos(row, Q4::EIGHTS * quarter + (j ^ v_turn)));
  }
  int page_next = -1;      // page of key `lane` of the next block to be asked for, read a block ahead of its use
  uint64_t seen_next = 0;  // keys of the block asked for last that exist
  Q4 kq, vq;
  auto look_up = [&](int base) __attribute__((always_inline)) {
    const int pos = base + lane;
    page_next = pos < k_end ? p.pv.pages[(int64_t)t.s * p.pv.pages_ld + (pos >> p.pv.page_shift)] : -1;
  };
  auto fetch = [&](int base) __attribute__((always_inline)) {
    seen_next = __ballot((uint32_t)page_next < (uint32_t)p.pv.num_pages);
    const int page = __shfl(page_next, row, 64), slot = (base + row) & ((1 << p.pv.page_shift) - 1);
    const bool ok = in && (uint32_t)page < (uint32_t)p.pv.num_pages;
    const int64_t off = page * p.pv.page_stride + slot * p.pv.slot_stride;
    const int64_t soff = page * p.scale_page + slot * p.scale_slot;
    const uint8_t* zero = (const uint8_t*)pq_zero;
    kq.load(ok ? kbase + off : zero, ok ? ksbase + soff : zero);
    vq.load(ok ? vbase + off : zero, ok ? vsbase + soff : zero);
  };

  const int lim_lo = t.limit(p, t.first / p.group);
  hidden[wave] = 0;
  const int n_blocks = uniform((k_end - k_begin + PA_KEYS - 1) / PA_KEYS);
  if (n_blocks > 0) {
    look_up(k_begin);
    fetch(k_begin);
    look_up(k_begin + PA_KEYS);
  }
  for (int j = 0; j < n_blocks; ++j) {
    const uint64_t seen = seen_next;
    const int base = k_begin + j * PA_KEYS;
    const uint32_t st = lds0 + (uint32_t)((j & 1) * STAGE);
    if (lim_lo < end && base + PA_KEYS > lim_lo && vq.hide()) hidden[wave] = 1;
    kq.swap(1, k_turn & 1), kq.swap(2, k_turn & 2);
    vq.swap(1, v_turn & 1), vq.swap(2, v_turn & 2);
#pragma unroll
    for (int i = 0; i < Q4::EIGHTS; ++i) {
      *(lds_u32x4_t*)(uintptr_t)(st + k_wr[i]) = kq.eight(i);
      *(lds_u32x4_t*)(uintptr_t)(st + v_wr[i]) = vq.eight(i);
    }
    if (j + 1 < n_blocks) {
      fetch(base + PA_KEYS);
      look_up(base + 2 * PA_KEYS);
    }
    lds_ring_barrier();  // everyone's share of block j is in place, and block j - 1 has been read
    if (wave_has_rows) rows.block(st, base, seen);
  }
  PqNan<D, BITS> nan(lds.few.table);
  if (n_blocks > 0 && (hidden[0] | hidden[1] | hidden[2] | hidden[3]))  // set before the last block's barrier
    nan.look(p, t, kvh, max(k_begin, lim_lo - PA_KEYS + 1), k_end, lds.few.table);
  if (wave_has_rows) rows.end(p, t, wave, n_packed, piece, whole, [&](int c) { return nan.seen(rows.lim, c); });
}

// A tile's keys in pieces, each a workgroup's; the order of the workgroups as in mi_paged.hip.
template <int D, int BITS>
__global__ void __launch_bounds__(64 * PF_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
    paged_attn_quant_few_kernel(QuantParams p) {
  __shared__ PqShared<D> lds;
  const int inner = p.n_kv * p.pieces, x = uniform(blockIdx.x / inner);
  const int at_inner = uniform((int)((blockIdx.x % inner + (uint32_t)x % p.pieces * p.n_kv) % inner));
  const int kvh = uniform(at_inner % p.n_kv), piece = uniform(at_inner / p.n_kv);
  const PaTile t = pa_tile(p, x);
  if (t.s < 0) return;
  const int end = t.end(p), plen = pa_piece(p, end);
  if (piece > 0 && (int64_t)piece * plen >= end) return;
  const int k_begin = piece * plen;
  pq_segment<D, BITS, false>(p, lds, t, kvh, k_begin, k_begin + min(plen, end - k_begin), plen >= end,
                      [&](int row, int head) { return ((int64_t)piece * p.pv.total_q + row) * p.n_heads + head; });
}

// The first blocks of a sequence arrive 4 us after the last sum of the one before, in which a workgroup does 300 keys:
// counted as 256, the workgroups end together (64 sequences of 500 to 8000 keys in 4 bits: 28.1 us, not counted 30.7, as 512
// 28.5; 16 in 8 bits 39, 40.6 and 38.2).
constexpr int PQ_EXTRA = 256 / PF_BLOCK;
template <int D, int BITS>
__global__ void __launch_bounds__(64 * PF_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
    paged_attn_quant_share_kernel(QuantParams p) {
  __shared__ PqShared<D> lds;
  __shared__ PfPrefix prefix;
  const int kvh = uniform(blockIdx.x % p.n_kv);
  pf_over_share<PQ_EXTRA>(p, prefix, uniform((int)(blockIdx.x / p.n_kv)),
                          [&](const PaTile& t, int k_begin, int k_end, bool whole, auto part_at) __attribute__((always_inline)) {
                            pq_segment<D, BITS, true>(p, lds, t, kvh, k_begin, k_end, whole, part_at);
                          });
}

template <int D, int BITS>
int pq_launch(const QuantParams& p, const PaPlan& plan, hipStream_t hs) {
  return pa_launch(
      p, plan, hs, [&](unsigned wgs) { paged_attn_quant_share_kernel<D, BITS><<<wgs, 64 * PF_WAVES, 0, hs>>>(p); },
      [&](unsigned wgs) { paged_attn_quant_few_kernel<D, BITS><<<wgs, 64 * PF_WAVES, 0, hs>>>(p); },
      [&](unsigned wgs) { paged_attn_quant_kernel<D, BITS><<<wgs, 256, 0, hs>>>(p); });
}

}  // namespace
}  // namespace mig

using namespace mig;

extern "C" {

size_t mi_paged_attn_quant_workspace_size(int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t n_seqs,
                                          int64_t total_q, int64_t max_q_len, int64_t max_kv_len) {
  return pa_workspace_size(n_heads, n_kv, head_dim, n_seqs, total_q, max_q_len, max_kv_len);
}

int mi_paged_attn_quant(void* stream, const void* Q, int64_t q_t, int64_t q_h, void* O, int64_t o_t, int64_t o_h,
                        float* lse, int64_t n_heads, const mi_quant_cache* cache, const mi_paged_seqs* seqs,
                        int64_t max_q_len, int64_t max_kv_len, int32_t causal, float scale, void* workspace,
                        size_t workspace_bytes) {
  int st = check_quant(cache, seqs);
  if (st != MI_OK) return st;
  QuantParams p;
  PaPlan plan;
  bool launch;
  st = pa_prepare(p, plan, launch, Q, q_t, q_h, O, o_t, o_h, lse, n_heads, cache->n_kv, cache->head_dim, cache->page_size,
                  seqs, paged_view(cache, seqs), max_q_len, max_kv_len, causal, scale, workspace, workspace_bytes);
  if (st != MI_OK || !launch) return st;
  p.k = cache->k, p.v = cache->v;
  p.ks = (const uint8_t*)cache->k_scale, p.vs = (const uint8_t*)cache->v_scale;
  p.scale_page = cache->scale_page_stride, p.scale_head = cache->scale_head_stride, p.scale_slot = cache->scale_slot_stride;
  hipStream_t hs = (hipStream_t)stream;
  const bool narrow = cache->head_dim <= 64;
  if (cache->format == MI_KV_E2M1) return narrow ? pq_launch<64, 4>(p, plan, hs) : pq_launch<128, 4>(p, plan, hs);
  return narrow ? pq_launch<64, 8>(p, plan, hs) : pq_launch<128, 8>(p, plan, hs);
}

}  // extern "C"
