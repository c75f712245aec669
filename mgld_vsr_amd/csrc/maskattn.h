// maskattn.h — what the masked-attention kernels (maskattn.hip: forward, maskattn_grad.hip: gradient) share: operand types, the LDS image of a
// tile, scores, visibility and the list of tiles that a group of query rows has to visit.
#pragma once
#include "common.h"

namespace {

typedef __bf16 bf16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char* ma_lds;

template <typename T> struct MaVec;
template <> struct MaVec<f16> { typedef f16x8 v8; };
template <> struct MaVec<bf16> { typedef bf16x8 v8; };
__device__ __forceinline__ f32x16 ma_mfma(const f16x8 a, const f16x8 b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 ma_mfma(const bf16x8 a, const bf16x8 b, const f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 ma_zero() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}
// eight fp32 values -> eight T, round to nearest even: the probabilities (and dS) become operands of the second product; their relative
// rounding error (2^-9 bf16, 2^-12 fp16) is independent per key and averages out over the sum, the sum itself stays fp32
template <typename T>
__device__ __forceinline__ typename MaVec<T>::v8 ma_pack(const float* x) {
  typename MaVec<T>::v8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (T)x[i];
  return r;
}
__device__ __forceinline__ constexpr int ma_row(const int r) { return (r & 3) + 8 * (r >> 2); }   // accumulator register -> row (+ 4 * lane half)

// keeps the compiler from carrying x + 0, x + 1, .. x + 31 around a loop in registers of their own
__device__ __forceinline__ int ma_opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

constexpr float MA_LOG2E = 1.44269504088896340736f, MA_LN2 = 0.69314718055994530942f;
#define MA_INF __builtin_inff()
constexpr int MA_KT = 64;          // keys (rows) per tile
__host__ __device__ inline int ma_tiles(const int n) { return (n + MA_KT - 1) / MA_KT; }
constexpr int MA_MAX_REACH = 1024; // a head's distance row lives in LDS,
constexpr int MA_PAD = 64;         // with its end values repeated this often
__host__ __device__ inline int ma_rel_floats(const int reach) { return 2 * reach + 1 + 2 * MA_PAD; }

// ---- LDS image of a [rows][D] tile: rows of 2 D bytes, 16-byte chunk c of row r at chunk c ^ swz(r).  Two kinds of reads:
// The swizzle moves consecutive rows (pairs of them at D = 64) by TWO chunks:
//  * row operand (rows r0 + lane % 32, eight consecutive d): one ds_read_b128, eight rows in eight different chunks;
//  * transposed operand (row d = dt * 32 + lane % 32, k = tile rows kb + 4 half + 0..3 and kb + 8 + 4 half + 0..3: the order in which
//    an accumulator holds its rows): two ds_read_b64_tr_b16, which hand lane i of 16 the four rows of column i of a [4][16] block; the
//    block's four 32-byte pieces lie in different banks (a swizzle by single chunks put two of them into the same ones).
template <int D>
struct Tile {
  static constexpr int RB = 2 * D;
  static constexpr int CH = D / 8;                       // 16-byte chunks per row
  __device__ static __forceinline__ int swz(const int r) { return D == 128 ? (r & 3) << 1 | ((r >> 2) & 1) | (r & 8) : (r & 2) | ((r >> 2) & 1) | (r & 8) >> 1; }
  __device__ static __forceinline__ int chunk_at(const int row, const int c) { return row * RB + ((c ^ swz(row)) << 4); }
  // lane's base for row operands; add (r0 * RB), XOR (ks * 32)
  __device__ static __forceinline__ int row_base(const int lane) { return (lane & 31) * RB + (((lane >> 5) ^ swz(lane & 31)) << 4); }
  // lane's base for transposed operands
  __device__ static __forceinline__ int tr_base(const int lane) {
    const int i = lane & 15, r = 4 * (lane >> 5) + (i >> 2), c = ((lane & 31) >> 4) * 2 + ((i & 3) >> 1);
    return r * RB + ((c ^ swz(r)) << 4) + (i & 1) * 8;
  }
  template <typename V8>
  __device__ static __forceinline__ V8 row_frag(const char* t, const int base, const int r0, const int ks) { return *(const V8*)(t + ((base ^ (ks * 32)) + r0 * RB)); }
  template <typename V8>
  __device__ static __forceinline__ V8 tr_frag(const char* t, const int base, const int dt, const int kb) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(ma_lds)(t + ((base ^ (dt * 64)) + kb * RB)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(ma_lds)(t + ((base ^ (dt * 64) ^ (D == 128 ? 128 : 64)) + (kb + 8) * RB)));
    const s16x8 r = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(V8, r);
  }
};

// A run of N matrix products whose operands come from LDS: operand i + AHEAD is requested before product i, in this order.  (Left alone the
// compiler reads each operand right before its product and waits out the LDS latency every time: 2.3 us per 64-key tile at d = 128.)
template <int I> struct MaIdx {
  static constexpr int value = I;
  constexpr operator int() const { return I; }
};
template <int I, int N, int AHEAD, typename V8, typename Read, typename Mul>
__device__ __forceinline__ void ma_stream_from(V8 (&ring)[AHEAD + 1], const Read& read, const Mul& mul) {
  if constexpr (I < N + AHEAD) {
    if constexpr (I < N) ring[I % (AHEAD + 1)] = read(MaIdx<I>{});
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (I >= AHEAD) mul(MaIdx<I - AHEAD>{}, ring[(I - AHEAD) % (AHEAD + 1)]);
    __builtin_amdgcn_sched_barrier(0);
    ma_stream_from<I + 1, N, AHEAD, V8>(ring, read, mul);
  }
}
template <int N, int AHEAD, typename V8, typename Read, typename Mul>
__device__ __forceinline__ void ma_stream(const Read read, const Mul mul) {
  V8 ring[AHEAD + 1];
  ma_stream_from<0, N, AHEAD, V8>(ring, read, mul);
}
// f(0), f(1), .. f(N - 1) with constant arguments
template <int I, int N, typename F>
__device__ __forceinline__ void ma_each(const F& f) {
  if constexpr (I < N) {
    f(MaIdx<I>{});
    ma_each<I + 1, N>(f);
  }
}

// ---- global -> LDS by DMA (`buffer_load_dwordx4 ... lds`: no staging registers, no ds_write pass).  A piece is 1 KiB of the image = 1024 / RB rows;
// lane l fills slot l of it and therefore fetches chunk (slot ^ swz(row)) of its row.  An offset past the descriptor's end delivers zeros:
// rows at or past `limit` (they may hold anything) and chunks past head_dim are sent there.  The base moves with the tile (64-bit), so an
// offset never passes 31 bits however long the tensor.  The instruction is written as asm so that the compiler does not drain the queue in front of
// the next LDS read; it has no output register, and the kernel waits (ma_dma_wait) before the barrier that hands the tile over.
#if defined(__HIP_DEVICE_COMPILE__)
typedef unsigned ma_rsrc __attribute__((ext_vector_type(4)));
__device__ __forceinline__ ma_rsrc ma_make_rsrc(const uint64_t a) {
  return ma_rsrc{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)) & 0xffffu, 0x7fffffffu, 0x00020000u};
}
// lane l's 16 bytes at base + voff + soff -> LDS bytes lds + 16 l (lds, base, soff wave-uniform; m0 is put back: the compiler takes it as its own)
__device__ __forceinline__ void ma_dma16(const unsigned lds, const unsigned voff, const ma_rsrc rs, const unsigned soff) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(lds), "v"(voff), "s"(rs), "s"(soff) : "memory");
}
// 64 consecutive 4-byte words (one per lane; words at or past `left` arrive as zeros)
__device__ __forceinline__ void ma_dma4(const unsigned lds, const int lane, const int left, const void* base) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(lane < left ? lane * 4u : 0x80000000u), "s"(ma_make_rsrc((uint64_t)base)) : "memory");
}
#else
typedef unsigned ma_rsrc;
__device__ __forceinline__ ma_rsrc ma_make_rsrc(const uint64_t) { return 0; }
__device__ __forceinline__ void ma_dma16(const unsigned, const unsigned, const ma_rsrc, const unsigned) {}
__device__ __forceinline__ void ma_dma4(const unsigned, const int, const int, const void*) {}
#endif
__device__ __forceinline__ void ma_dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// in front of a loop over tiles, told to the compiler: the block's own loads have landed.  (Where it cannot see that, it waits for the whole queue inside the loop, and so for
// the next tile's DMA: 61 -> 68 us on 2 x 2048 tokens, 16 / 4 heads of 128.)
__device__ __forceinline__ void ma_loads_landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt(0) alone
__device__ __forceinline__ unsigned ma_lds_addr(const void* s) { return (unsigned)(uintptr_t)(ma_lds)s; }

// ROWS x D tile of one matrix, moved by NW waves: this wave's pieces.  With four waves a wave's pieces lie 16 or 32 rows apart, where the swizzle
// repeats: one lane offset serves all of them and the scalar offset moves.
template <int D, int ROWS, int NW>
struct TileDma {
  static constexpr int RPP = 1024 / Tile<D>::RB, NP = ROWS / RPP / NW, STEP = NW * RPP;
  static constexpr bool SAME = STEP % 16 == 0;
  unsigned voff[SAME ? 1 : NP];
  int row0;
  unsigned lds;             // byte offset of this wave's first piece in the tile
  __device__ TileDma(const int wave, const int lane, const int64_t stride, const int head_dim) {
    row0 = wave * RPP + lane / Tile<D>::CH;
#pragma unroll
    for (int j = 0; j < (SAME ? 1 : NP); ++j) {
      const int row = row0 + j * STEP, c = (lane % Tile<D>::CH) ^ Tile<D>::swz(row);
      voff[j] = c * 8 < head_dim ? (unsigned)(SAME ? row : row0) * (unsigned)(stride * 2) + c * 16 : 0x80000000u;
    }
    lds = __builtin_amdgcn_readfirstlane(wave) * 1024;
  }
  // the ROWS rows (stride elements apart) that begin first_byte into the matrix at `base` -> the tile at LDS byte address `tile`; rows at or past
  // `left` and rows that gone() names arrive as zeros (gone is asked only if `some`)
  template <typename Gone>
  __device__ __forceinline__ void load(const void* base, const int64_t first_byte, const int64_t stride, const int left, const unsigned tile, const bool some,
                                       const Gone gone) const {
    const ma_rsrc rs = ma_make_rsrc((uint64_t)base + (uint64_t)first_byte);
    const unsigned step = __builtin_amdgcn_readfirstlane((int)((unsigned)stride * (2 * STEP))), to = __builtin_amdgcn_readfirstlane((int)(tile + lds));
    bool ok[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) ok[j] = row0 + j * STEP < left;
    if (some) {
#pragma unroll
      for (int j = 0; j < NP; ++j) ok[j] = ok[j] && !gone(row0 + j * STEP);
    }
#pragma unroll
    for (int j = 0; j < NP; ++j) ma_dma16(to + j * NW * 1024, ok[j] ? voff[SAME ? 0 : j] : 0x80000000u, rs, j * step);
  }
  __device__ __forceinline__ void load(const void* base, const int64_t first_byte, const int64_t stride, const int left, const unsigned tile) const {
    load(base, first_byte, stride, left, tile, false, [](int) { return false; });
  }
};

// ---- scores, in log2 units (a probability is one subtraction and one exp2).  Cap: u = cap tanh(t / cap) = cap (1 - 2 / (1 + e^(2 t / cap))):
//  squash = -1 / (1 + exp2(q.k * pre)), one exp2 and one reciprocal per score, u = cap (1 + 2 squash).  That is off by up to 2^-23 of the CAP, whatever the
//  score: 2^-16 at a cap of 128, and at 1e8 nothing of an ordinary score is left.  Above MA_WIDE_CAP (MODE bit MA_WIDE) scores below a quarter of the cap therefore take
//  tanh's odd series, u = t (1 - x^2 / 3 + 2 x^4 / 15 - 17 x^6 / 315 + 62 x^8 / 2835), x = t / cap < 1/4 (the next term is 2^-26), and the others 1 - 2 / (1 + e^2x),
//  whose error is then 2^-21 of u: relative in both.  It costs nine more instructions per score, so small caps keep the short form: 8192 causal tokens, 32 / 8 heads of
//  128 bf16, 740 us against 893; 4096 tokens, 16 heads of 64 fp16, 118 against 174; the gradient of 4096 / 2048 such tokens 1042 against 1241, 228 against 279.
constexpr int MA_CAP = 1, MA_SLOPES = 2, MA_REL = 4, MA_WIDE = 8;       // MODE bits; slopes and distance rows exclude each other; wide: with a cap
constexpr float MA_WIDE_CAP = 128.f;
// tanh(x) / x, x^2 = s <= 1/16
__device__ __forceinline__ float ma_tanh_ratio(const float s) {
  return fmaf(s, fmaf(s, fmaf(s, fmaf(s, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
}
template <int MODE>
struct Score {
  static constexpr bool CAP = MODE & MA_CAP, SLOPES = MODE & MA_SLOPES, REL = MODE & MA_REL, WIDE = MODE & MA_WIDE, BIAS = SLOPES || REL;
  float pre, capA, slope2, scale2;
  const float* rel;          // LDS: the head's distance row in log2 units, distance 0 at index reach + MA_PAD
  int reach;
  __device__ Score(const MgldMaskAttn& p, const int h, const float* srel) {
    pre = CAP ? fminf(2.f * MA_LOG2E * p.scale / p.softcap, 3.4e38f) : p.scale * MA_LOG2E;       // (finite: a score of zero is zero under the smallest cap too)
    capA = CAP ? (WIDE ? 1.f : 2.f) * MA_LOG2E * p.softcap : 0.f;
    scale2 = p.scale * MA_LOG2E;
    slope2 = SLOPES ? p.slopes[h] * MA_LOG2E : 0.f;
    reach = p.reach;
    rel = srel + reach + MA_PAD;
  }
  // the bias of a lane's 16 scores of a 32 x 32 block: those at distance delta + off (UP) or delta - off, off = ma_row(0 .. 15) < 32.  The distance
  // row goes on for MA_PAD entries past both ends, so one clamp of the lane's first distance serves all 16 reads (immediate offsets).
  struct At { const float* tab; float d; };
  template <bool UP>
  __device__ __forceinline__ At at(const int delta) const {
    At a{nullptr, 0.f};
    if (SLOPES) a.d = (float)delta;
    if (REL) a.tab = rel + (UP ? min(max(delta, 1 - MA_PAD - reach), reach + MA_PAD - 32) : min(max(delta, 32 - MA_PAD - reach), reach + MA_PAD - 1) - 31);
    return a;
  }
  __device__ __forceinline__ float squash(const float acc) const { return -__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(acc * pre)); }   // in [-1, 0]
  // wide: u in log2 units, and tanh
  __device__ __forceinline__ float bend(const float acc, float& th) const {
    const float a = acc * pre, x = a * (0.5f * MA_LN2), r = ma_tanh_ratio(x * x);
    const bool near = fabsf(x) < 0.25f;
    const float far = fmaf(2.f, squash(acc), 1.f);
    th = near ? x * r : far;
    return near ? acc * scale2 * r : capA * far;
  }
  template <bool UP>
  __device__ __forceinline__ float raised(const float u, const At a, const int off) const {      // u + bias
    if (SLOPES) return fmaf(-slope2, fabsf(UP ? a.d + (float)off : a.d - (float)off), u);
    return REL ? u + a.tab[UP ? off : 31 - off] : u;
  }
  // the cap's slope, 1 - tanh^2, from what prob() left
  __device__ __forceinline__ float slope(const float sq) const { return WIDE ? fmaf(-sq, sq, 1.f) : -4.f * sq * (1.f + sq); }       // (tanh = 1 + 2 squash)
  // score in log2 units from the scaled one
  template <bool UP>
  __device__ __forceinline__ float biased(const float f, const float x, const float c, const At a, const int off) const {      // f x + c + bias
    if (SLOPES) return fmaf(-slope2, fabsf(UP ? a.d + (float)off : a.d - (float)off), CAP ? fmaf(f, x, c) : f * x);
    if (REL) return CAP ? fmaf(f, x, c + a.tab[UP ? off : 31 - off]) : fmaf(f, x, a.tab[UP ? off : 31 - off]);
    return 0.f;
  }
  __device__ __forceinline__ float score(const float acc, const At a, const int off) const {
    if (WIDE) {
      float th;
      const float u = bend(acc, th);
      return raised<true>(u, a, off);
    }
    if (!BIAS) return CAP ? fmaf(squash(acc), capA, 0.5f * capA) : acc * pre;
    return biased<true>(CAP ? squash(acc) : acc, CAP ? capA : pre, 0.5f * capA, a, off);
  }
  // P = 2^(score - lse2); sq: the squashed dot product (wide: tanh), for slope()
  template <bool UP>
  __device__ __forceinline__ float prob(const float acc, const At a, const int off, const float lse2, float& sq) const {
    if (WIDE) {
      const float u = bend(acc, sq);
      return __builtin_amdgcn_exp2f(raised<UP>(u, a, off) - lse2);
    }
    sq = CAP ? squash(acc) : 0.f;
    if (!BIAS) return __builtin_amdgcn_exp2f(CAP ? sq * capA + (0.5f * capA - lse2) : acc * pre - lse2);
    return __builtin_amdgcn_exp2f(biased<UP>(CAP ? sq : acc, CAP ? capA : pre, 0.5f * capA, a, off) - lse2);
  }
};

// ---- what a batch row lets its queries see
struct BatchSpan {
  int len, pos0, prefix;
  __device__ BatchSpan(const MgldMaskAttn& p, const int b) {
    len = p.kv_len ? min(max(p.kv_len[b], 0), p.Nkv) : p.Nkv;
    pos0 = p.q_from_end ? len - p.Nq : p.q_pos0;
    prefix = p.prefix ? p.prefix[b] : 0;
  }
  // keys below this index are in sight of position pos (documents aside)
  __device__ __forceinline__ int limit(const MgldMaskAttn& p, const int pos) const {
    return p.causal ? min(len, max(pos < 0x7fffffff ? pos + 1 : pos, prefix)) : len;
  }
};

// a group of consecutive query rows [i0, i0 + n): its limits and the range of its document numbers
struct RowGroup {
  int lim_min, lim_max;       // smallest / largest limit() over the rows
  int dmin, dmax;             // over rows with a document; dmin > dmax: none
  bool uniform;               // every row has the same document
};
// documents of rows [i0, i1), reduced over the wave (all lanes call); ids: this batch row's numbers
__device__ __forceinline__ bool ma_doc_range(const int32_t* ids, const int i0, const int i1, int& dmin, int& dmax, bool& uniform) {
  int lo = 0x7fffffff, hi = -1, neg = 0;
  for (int i = i0 + (int)(threadIdx.x & 63); i < i1; i += 64) {
    const int v = ids[i];
    if (v >= 0) { lo = min(lo, v); hi = max(hi, v); } else neg = 1;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o, 64));
    hi = max(hi, __shfl_xor(hi, o, 64));
    neg |= __shfl_xor(neg, o, 64);
  }
  dmin = lo; dmax = hi; uniform = !neg && lo == hi;
  return neg != 0;
}
__device__ __forceinline__ RowGroup ma_row_group(const MgldMaskAttn& p, const BatchSpan& bs, const int b, const int i0, const int n) {
  RowGroup g;
  const int i1 = min(i0 + n, p.Nq);
  g.lim_min = bs.limit(p, bs.pos0 + i0);
  g.lim_max = i1 > i0 ? bs.limit(p, bs.pos0 + i1 - 1) : 0;
  g.dmin = 0; g.dmax = -1; g.uniform = false;
  if (p.doc_q) ma_doc_range(p.doc_q + b * p.doc_q_sb, i0, i1, g.dmin, g.dmax, g.uniform);
  return g;
}

// document numbers of the 64-row tiles, written by ma_doc_tiles_kernel: {min, max, all 64 rows in one document, some row without}
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// which tiles of [t0, t0 + 64) the group has to visit (act), and in which of them it sees every pair (full); lane l judges tile t0 + l
__device__ __forceinline__ void ma_window(const MgldMaskAttn& p, const RowGroup& g, const i32x4 dt, const int t, unsigned long long& act,
                                          unsigned long long& full) {
  const int64_t k0 = (int64_t)t * MA_KT;
  bool a = k0 < g.lim_max, f = k0 + MA_KT <= g.lim_min;
  if (p.doc_q) {
    a = a && dt[0] <= g.dmax && dt[1] >= g.dmin;
    f = f && dt[2] && g.uniform && dt[0] == g.dmin;
  }
  act = __ballot(a);
  full = __ballot(a && f);
}

// the distance rows of heads h .. h + n - 1 into LDS, in log2 units (all threads of the block; a barrier follows in the caller)
__device__ __forceinline__ void ma_load_rel(const MgldMaskAttn& p, const int h, const int n, float* srel) {
  const int w = ma_rel_floats(p.reach), nr = 2 * p.reach + 1;
  for (int x = threadIdx.x; x < n * w; x += blockDim.x) {
    const int g = x / w, e = x - g * w;
    srel[x] = p.rel[(int64_t)(h + g) * nr + min(max(e - MA_PAD, 0), nr - 1)] * MA_LOG2E;
  }
}

// ---- exact row by row, for the few rows whose fast result is not finite: a product with a zero probability turns an infinity or NaN of a
// value (gradient: a key) that the row does not see into NaN.  One wave recomputes row (b, h, i) from its visible keys alone: lanes are keys for the scores,
// then elements of d for the sum.
// The kernel's first argument as the rare rows read it: through a pointer that the compiler cannot look behind, so that their two dozen values are loaded
// there and do not sit in scalar registers (spilled to vector lanes) through the whole kernel: 728 -> 704 us on 8192 causal tokens, 32 / 8 heads of 128,
// cap 50.  (The forward at d = 64 has no registers to load them into.)
__device__ __forceinline__ const MgldMaskAttn& ma_late_args() {
#if defined(__HIP_DEVICE_COMPILE__)
  uint64_t a = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const MgldMaskAttn*)(const __attribute__((address_space(4))) void*)a;
#else
  return *(const MgldMaskAttn*)nullptr;
#endif
}
template <typename T>
struct ExactRow {
  const MgldMaskAttn& p;
  const T *q, *kb, *vb;
  const int32_t* ids;        // the keys' document numbers
  int b, h, i, d, pos, lim, doc;
  __device__ ExactRow(const MgldMaskAttn& pp, const int bb, const int hh, const int ii) : p(pp), b(bb), h(hh), i(ii), d(pp.head_dim) {
    const BatchSpan bs(p, b);
    const int hk = h / (p.heads / p.kv_heads);
    pos = bs.pos0 + i;
    lim = bs.limit(p, pos);
    doc = p.doc_q ? p.doc_q[b * p.doc_q_sb + i] : 0;
    ids = p.doc_k ? p.doc_k + b * p.doc_k_sb : nullptr;
    q = (const T*)p.Q + b * p.q_sb + (int64_t)i * p.q_si + h * p.q_sh;
    kb = (const T*)p.K + b * p.k_sb + hk * p.k_sh;
    vb = (const T*)p.V + b * p.v_sb + hk * p.v_sh;
  }
  __device__ __forceinline__ bool seen(const int j) const { return j < lim && doc >= 0 && !(ids && ids[j] != doc); }
  // of a key that the row sees: the score in log2 units, and the cap's slope there
  __device__ __forceinline__ float score(const int j, float& slope) const {
    const T* k = kb + (int64_t)j * p.k_si;
    float t = 0.f;
    for (int e = 0; e < d; ++e) t += (float)q[e] * (float)k[e];
    t *= p.scale;
    slope = 1.f;
    if (p.softcap > 0.f) {
      const float x = t / p.softcap;
      const bool near = fabsf(x) < 0.25f;
      const float r = ma_tanh_ratio(x * x), th = near ? x * r : 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * (2.f * MA_LOG2E)));
      t = near ? t * r : p.softcap * th;
      slope = 1.f - th * th;
    }
    const int delta = j - pos;
    if (p.slopes) t -= p.slopes[h] * fabsf((float)delta);
    if (p.rel) t += p.rel[(int64_t)h * (2 * p.reach + 1) + min(max(delta, -p.reach), p.reach) + p.reach];
    return t * MA_LOG2E;
  }
  // sum over the keys of [j0, j0 + 64) that are seen of w (lane's key j0 + lane) times their rows at `rows`: a lane's elements lane, lane + 64
  __device__ __forceinline__ void add(const int j0, const float w, const bool s, const T* rows, const int64_t stride, float& a0, float& a1) const {
    const int lane = threadIdx.x & 63;
    unsigned long long todo = __ballot(s);
    while (todo) {
      const int c = __builtin_ctzll(todo);
      todo &= todo - 1;
      const float wc = __shfl(w, c, 64);
      const T* r = rows + (int64_t)(j0 + c) * stride;
      if (lane < d) a0 += wc * (float)r[lane];
      if (lane + 64 < d) a1 += wc * (float)r[lane + 64];
    }
  }
  __device__ __forceinline__ T* at(void* out, const int64_t sb, const int64_t si, const int64_t sh) const { return (T*)out + b * sb + (int64_t)i * si + h * sh; }
  __device__ __forceinline__ void put(void* out, const int64_t sb, const int64_t si, const int64_t sh, const float a0, const float a1) const {
    const int lane = threadIdx.x & 63;
    T* const o = at(out, sb, si, sh);
    if (lane < d) o[lane] = (T)a0;
    if (lane + 64 < d) o[lane + 64] = (T)a1;
  }
};
// Is the row's fast result, stored at `out`, not finite only where a row of `rows` (V for o, K for dQ) that it sees is not finite either, in the same column?  Then it stands:
// in a run that diverged every row is one of these (4096 tokens, 32 / 8 heads of 128: 223 ms without this look, which mostly ends at its first rows).  A NaN of o needs a NaN,
// an infinity an infinity (the weights are positive); dQ's weights may be zero or of either sign, so there one does for the other.
template <typename T>
__device__ __forceinline__ bool ma_stands(const ExactRow<T>& row, const T* rows, const int64_t stride, const T* out, const bool either) {
  constexpr unsigned EXP = __is_same(T, f16) ? 0x7c00u : 0x7f80u;      // magnitude bits: of infinity; above: NaN
  const int lane = threadIdx.x & 63;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");              // (the wave's own stores are read back)
  auto mag = [&](const T* x, const int c) __attribute__((always_inline)) { return lane + 64 * c < row.d ? ((const unsigned short*)x)[lane + 64 * c] & 0x7fffu : 0u; };
  const unsigned o0 = mag(out, 0), o1 = mag(out, 1), t0 = o0 > EXP && !either ? EXP + 1 : EXP, t1 = o1 > EXP && !either ? EXP + 1 : EXP;
  bool ok0 = o0 < EXP, ok1 = o1 < EXP;
  for (int j0 = 0; j0 < row.lim; j0 += 8) {
    unsigned top = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const T* const x = rows + (int64_t)min(j0 + u, row.lim - 1) * stride;
      top = max(top, max(mag(x, 0), mag(x, 1)));
    }
    if (!__any(top >= EXP)) continue;
    const int j1 = min(j0 + 8, row.lim);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      if (!row.seen(j)) continue;
      const T* const x = rows + (int64_t)j * stride;
      ok0 = ok0 || mag(x, 0) >= t0;
      ok1 = ok1 || mag(x, 1) >= t1;
    }
    if (__all(ok0 && ok1)) return true;
  }
  return false;
}
template <typename T>
__device__ __forceinline__ void ma_slow_row(const MgldMaskAttn& p, const int b, const int h, const int i) {
  const ExactRow<T> row(p, b, h, i);
  if (ma_stands(row, row.vb, p.v_si, (const T*)row.at(p.O, p.o_sb, p.o_si, p.o_sh), false)) return;
  const int lane = threadIdx.x & 63;
  float m = -MA_INF, sl;
  for (int j = lane; j < row.lim; j += 64)
    if (row.seen(j)) m = fmaxf(m, row.score(j, sl));
  m = wave_max(m);
  if (m == -MA_INF) m = 0.f;
  float l = 0.f, a0 = 0.f, a1 = 0.f;
  for (int j0 = 0; j0 < row.lim; j0 += 64) {
    const bool s = row.seen(j0 + lane);
    const float pr = s ? __builtin_amdgcn_exp2f(row.score(j0 + lane, sl) - m) : 0.f;
    l += pr;
    row.add(j0, pr, s, row.vb, p.v_si, a0, a1);
  }
  l = wave_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  row.put(p.O, p.o_sb, p.o_si, p.o_sh, a0 * inv, a1 * inv);
}
// dQ of the row, from its lse (log2 units) and D
template <typename T>
__device__ __forceinline__ void ma_slow_dq(const MgldMaskAttn& p, const int b, const int h, const int i, const float lse2, const float delta) {
  const ExactRow<T> row(p, b, h, i);
  const int lane = threadIdx.x & 63;
  if (ma_stands(row, row.kb, p.k_si, (const T*)row.at(p.dQ, p.dq_sb, p.dq_si, p.dq_sh), true)) return;
  const T* const g = (const T*)p.dO + b * p.do_sb + (int64_t)i * p.do_si + h * p.do_sh;
  float a0 = 0.f, a1 = 0.f;
  for (int j0 = 0; j0 < row.lim; j0 += 64) {
    const int j = j0 + lane;
    const bool s = row.seen(j);
    float dt = 0.f;
    if (s) {
      const T* v = row.vb + (int64_t)j * p.v_si;
      float dp = 0.f, sl;
      for (int e = 0; e < row.d; ++e) dp += (float)g[e] * (float)v[e];
      dt = __builtin_amdgcn_exp2f(row.score(j, sl) - lse2) * (dp - delta) * sl;
    }
    row.add(j0, dt, s, row.kb, p.k_si, a0, a1);
  }
  row.put(p.dQ, p.dq_sb, p.dq_si, p.dq_sh, a0 * p.scale, a1 * p.scale);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------------
// document tiles of keys, then of queries
inline int64_t ma_doc_bytes(const MgldMaskAttn* p) {
  return p->doc_q ? ((int64_t)p->batch * (ma_tiles(p->Nkv) + ma_tiles(p->Nq))) * 16 : 0;
}

}  // namespace

inline int ma_mode(const MgldMaskAttn* p) { return (p->softcap > 0.f ? MA_CAP : 0) | (p->softcap > MA_WIDE_CAP ? MA_WIDE : 0) | (p->slopes ? MA_SLOPES : 0) | (p->rel ? MA_REL : 0); }
// calls launch<T, D, MODE>(p, st) for the problem's type, head size and score form
#define MA_DISPATCH_MODE(launch, T, D, p, st)                                        \
  switch (ma_mode(p)) {                                                              \
    case 0: return launch<T, D, 0>(*p, st);                                          \
    case MA_CAP: return launch<T, D, MA_CAP>(*p, st);                                \
    case MA_SLOPES: return launch<T, D, MA_SLOPES>(*p, st);                          \
    case MA_SLOPES | MA_CAP: return launch<T, D, MA_SLOPES | MA_CAP>(*p, st);        \
    case MA_REL: return launch<T, D, MA_REL>(*p, st);                                \
    case MA_REL | MA_CAP: return launch<T, D, MA_REL | MA_CAP>(*p, st);              \
    case MA_WIDE | MA_CAP: return launch<T, D, MA_WIDE | MA_CAP>(*p, st);            \
    case MA_WIDE | MA_SLOPES | MA_CAP: return launch<T, D, MA_WIDE | MA_SLOPES | MA_CAP>(*p, st); \
    default: return launch<T, D, MA_WIDE | MA_REL | MA_CAP>(*p, st);                 \
  }
#define MA_DISPATCH(launch, p, st)                                                   \
  if (p->bf16) {                                                                     \
    if (p->head_dim <= 64) { MA_DISPATCH_MODE(launch, bf16, 64, p, st) }             \
    MA_DISPATCH_MODE(launch, bf16, 128, p, st)                                       \
  }                                                                                  \
  if (p->head_dim <= 64) { MA_DISPATCH_MODE(launch, f16, 64, p, st) }                \
  MA_DISPATCH_MODE(launch, f16, 128, p, st)

int ma_check(const MgldMaskAttn* p, bool grad);
int ma_doc_tiles(const MgldMaskAttn& p, void* out, hipStream_t st);
