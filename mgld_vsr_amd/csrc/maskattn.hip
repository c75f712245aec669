// maskattn.hip — attention with capped scores, distance biases and causal / prefix / document / length masks: forward.
//
//   s = [softcap tanh(./softcap)](scale q.k) + bias(j - p_i),  o = sum_visible softmax(s) v,  lse = log sum_visible exp s
//
// Two kernels: many query rows (one block per 128 rows of a head) and few rows over many keys (keys split over the grid, joined afterwards).
//  * Scores are computed transposed, S^T = K Q^T (v_mfma_f32_32x32x16): a lane holds 16 keys of ONE query row per 32-key half tile, so the row
//    maximum and sum are lane-local plus one exchange with lane ^ 32, and the probabilities are the second product's operand as they lie,
//    O^T = V^T P^T.  V stays row-major in LDS; its transposed fragments come from ds_read_b64_tr_b16.
//  * One pass with the running maximum (it moves only when a score exceeds it by 2^6, so the accumulator is rarely rescaled) and the sum in fp32.  In fp16
//    probabilities are held as 2^9 P <= 2^15: of many small ones beside a large one each is off by at most 2^-34 of it (as P, by 2^-25: half of the sum of
//    2^17 keys at 2^-24.6).
//  * Which tiles a block visits, and which of them need no mask, is decided 64 tiles at a time: lane l judges tile t0 + l and two
//    ballots give the bit masks.  A causal, prefix, length or document mask costs skipped tiles nothing and full tiles nothing.
//
// Bounds and figures (4 d products per visible pair; a large matrix product reaches 1400 TFLOP/s):
//  * many rows, d = 128: 880-905 TFLOP/s on full tiles, 750-780 under a cap (three transcendentals per score), ~740 at d = 64; ~10 us a launch beside that.
//    8192 tokens, 32 / 8 heads of 128, causal, cap 50: 697 us.  Neither pipe is full there: the vector pipe is active 72 % of the cycles, the matrix pipe 35 %, and waves
//    wait 21 % of theirs: the chain from a score over its exponentials to the second product, with two waves per SIMD to hide it.  128 rows a block =
//    two blocks per CU (three at d = 64), so one's barrier is the other's work.
//    Keeping unscaled scores (32 of 340 vector instructions fewer per tile) gained 0.8 % and spilled at d = 64; one m0 write for several DMA pieces: nothing.
//  * few rows: HBM.  16 sequences of up to 32768 cached tokens, 8 key heads of 128 (1.40 GB): 241 + 5 us, 5.6 TB/s.
#include "maskattn.h"

namespace {

// {min, max document number >= 0, all 64 rows in one document, some row without} of each 64-row tile: keys' tiles of every batch row, then the queries'
__global__ __launch_bounds__(64) void ma_doc_tiles_kernel(const int32_t* dk, const int32_t* dq, const int64_t k_sb, const int64_t q_sb, const int Nkv,
                                                          const int Nq, const int batch, i32x4* out) {
  const int ntk = (Nkv + MA_KT - 1) / MA_KT, ntq = (Nq + MA_KT - 1) / MA_KT;
  const int b = blockIdx.y;
  int t = blockIdx.x;
  const bool isq = t >= ntk;
  if (isq) t -= ntk;
  const int i0 = t * MA_KT, n = isq ? Nq : Nkv;
  int lo, hi;
  bool uni;
  const bool pad = ma_doc_range(isq ? dq + b * q_sb : dk + b * k_sb, i0, min(i0 + MA_KT, n), lo, hi, uni);
  if (threadIdx.x == 0) {
    const i32x4 r = {lo, hi, (int)(uni && i0 + MA_KT <= n), (int)pad};
    (isq ? out + (int64_t)batch * ntk + (int64_t)b * ntq : out + (int64_t)b * ntk)[t] = r;
  }
}

// a query row's running maximum (log2 units), sum and accumulators
constexpr float MA_SLACK = 6.f;        // the maximum moves when a score exceeds it by this much: probabilities stay below 2^6
template <typename T, int DT>
struct RowState {
  static constexpr float LIFT = __is_same(T, f16) ? 9.f : 0.f;       // probabilities are held as 2^LIFT P
  f32x16 o[DT];
  float m, l;
  __device__ RowState() : m(-MA_INF), l(0.f) {
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = ma_zero();
  }
  // the row's new scores reach mx (in this lane's half of the keys)
  __device__ __forceinline__ void rise(float mx) {
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__any(mx > m + MA_SLACK)) {                  // m = -inf: true as soon as something is visible
      const float mn = mx > m + MA_SLACK ? mx : m;
      const float al = m == -MA_INF ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= al;
      m = mn;
    }
  }
  __device__ __forceinline__ float base() const { return m == -MA_INF ? 0.f : m - LIFT; }
  __device__ __forceinline__ float unit() const { return m - LIFT; }       // what o and l are relative to (-inf: nothing was visible)
};

// masks a 32-key half of the scores: keys k0 + ma_row(r) + 4 half at or past `lim`, or of another document than dq
template <bool DOCS>
__device__ __forceinline__ void ma_mask(float* st, const int k0, const int lhi, const int lim, const int* sdoc, const int dq) {
  const int left = ma_opaque(lim - k0 - lhi * 4);
#pragma unroll
  for (int rg = 0; rg < 4; ++rg) {                     // registers 4 rg .. + 3: four consecutive keys
    const int j = rg * 8 + lhi * 4;
    i32x4 dk = {dq, dq, dq, dq};
    if (DOCS) dk = *(const i32x4*)(sdoc + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool vis = (rg * 8 + e < left) & (dk[e] == dq);
      st[rg * 4 + e] = vis ? st[rg * 4 + e] : -MA_INF;
    }
  }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------------------
// block: 4 waves x 32 query rows of one head; K / V tiles of 64 keys go by DMA into two LDS buffers each, K one tile ahead of V, one barrier per
// tile.  A wave computes the scores of tile t + 1 while it turns those of tile t into probabilities.
template <typename T, int D, int MODE>
__global__ __launch_bounds__(256, D == 64 && !((MODE & MA_CAP) && MODE != MA_CAP) ? 3 : 2) void ma_fwd_kernel(const MgldMaskAttn p, const i32x4* __restrict__ kdoc, const int nqb) {
  typedef typename MaVec<T>::v8 v8;
  typedef Tile<D> TL;
  constexpr int DK = D / 16, DT = D / 32;
  constexpr int TBYTES = MA_KT * TL::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];              // [2] x {K, V}, then doc numbers [2][64], then the distance row
  int* const sdoc = (int*)(smem + 4 * TBYTES);
  float* const srel = (float*)(sdoc + 2 * MA_KT);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lhi = lane >> 5;

  // block -> (batch row, head, row block).  Blocks go round-robin to the 8 XCDs: XCD x takes consecutive heads (which share K and V, and the L2),
  // all of them at one row block before the next; the last row blocks (the longest under a causal mask) come first.
  const int nbh = p.batch * p.heads;
  int bh, qb;
  if (nbh % 8 == 0) {
    const int per = nbh / 8, x = blockIdx.x & 7, j = blockIdx.x >> 3;
    bh = x * per + j % per;
    qb = nqb - 1 - j / per;
  } else {
    bh = blockIdx.x % nbh;
    qb = nqb - 1 - blockIdx.x / nbh;
  }
  const int b = bh / p.heads, h = bh % p.heads, hk = h / (p.heads / p.kv_heads);
  const int i0 = qb * 128, iw = i0 + wave * 32;
  const BatchSpan bs(p, b);
  const RowGroup gb = ma_row_group(p, bs, b, i0, 128), gw = ma_row_group(p, bs, b, iw, 32);
  const bool docs = p.doc_q != nullptr;
  const int ntk = (p.Nkv + MA_KT - 1) / MA_KT;
  if (docs) kdoc += (int64_t)b * ntk;

  const T* __restrict__ Qp = (const T*)p.Q + b * p.q_sb + h * p.q_sh;
  const T* __restrict__ Kp = (const T*)p.K + b * p.k_sb + hk * p.k_sh;
  const T* __restrict__ Vp = (const T*)p.V + b * p.v_sb + hk * p.v_sh;
  const int d8 = p.head_dim / 8;
  v8 zero;
#pragma unroll
  for (int i = 0; i < 8; ++i) zero[i] = (T)0.f;

  const int i = iw + l31;
  const int pos = bs.pos0 + i;
  const int dq = docs && i < p.Nq ? p.doc_q[b * p.doc_q_sb + i] : -1;
  const int lim = i < p.Nq && (!docs || dq >= 0) ? bs.limit(p, pos) : 0;         // a row without document sees nothing: its number (any negative one) may be a key's
  v8 qf[DK];
#pragma unroll
  for (int ks = 0; ks < DK; ++ks) qf[ks] = i < p.Nq && ks * 2 + lhi < d8 ? *(const v8*)(Qp + (int64_t)i * p.q_si + ks * 16 + lhi * 8) : zero;
  if (MODE & MA_REL) ma_load_rel(p, h, 1, srel);
  const Score<MODE> sc(p, h, srel);

  // tiles to visit
  const int nt = ma_tiles(gb.lim_max);
  int w0 = -64;
  unsigned long long bact = 0, wact = 0, wfull = 0, bfull = 0, pads = 0;
  auto advance = [&](int& flags) __attribute__((always_inline)) {      // next tile of the block, or -1; flags: 1 the wave visits it, 2 without mask, 4 padding rows
    while (!bact) {
      w0 += 64;
      if (w0 >= nt) return -1;
      const i32x4 dt = docs && w0 + lane < ntk ? kdoc[w0 + lane] : i32x4{0x7fffffff, -1, 0, 0};
      ma_window(p, gb, dt, w0 + lane, bact, bfull);
      ma_window(p, gw, dt, w0 + lane, wact, wfull);
      pads = __ballot(dt[3] != 0);
    }
    const int c = __builtin_ctzll(bact);
    bact &= bact - 1;
    flags = (int)((wact >> c) & 1) | (int)((wfull >> c) & 1) << 1 | (int)((pads >> c) & 1) << 2;
    return w0 + c;
  };

  const TileDma<D, MA_KT, 4> dk(wave, lane, p.k_si, p.head_dim), dv(wave, lane, p.v_si, p.head_dim);
  const unsigned lds0 = ma_lds_addr(smem);
  auto load_k = [&](const int t, const int buf, const int flags) __attribute__((always_inline)) {
    const int k0 = t * MA_KT;
    const int32_t* const ids = docs ? p.doc_k + b * p.doc_k_sb + k0 : nullptr;
    dk.load(Kp, (int64_t)k0 * p.k_si * 2, p.k_si, bs.len - k0, lds0 + buf * TBYTES, flags & 4, [&](const int r) { return ids[r] < 0; });
    if (docs && wave == 0) ma_dma4(lds0 + 4 * TBYTES + buf * MA_KT * 4, lane, bs.len - k0, ids);      // (zeros past the length: `lim` hides them)
  };
  auto load_v = [&](const int t, const int buf, const int flags) __attribute__((always_inline)) {
    const int k0 = t * MA_KT;
    const int32_t* const ids = docs ? p.doc_k + b * p.doc_k_sb + k0 : nullptr;
    dv.load(Vp, (int64_t)k0 * p.v_si * 2, p.v_si, bs.len - k0, lds0 + (2 + buf) * TBYTES, flags & 4, [&](const int r) { return ids[r] < 0; });
  };

  RowState<T, DT> rs;
  const int kbase = TL::row_base(lane), vbase = TL::tr_base(lane);
  constexpr int NP = 2 * DK, EPP = 32 / NP;            // products of a 64-key tile (scores, and P V as many), scores per product
  constexpr bool LATE = D == 128 && (MODE & MA_WIDE) && (MODE & (MA_REL | MA_SLOPES));       // the next scores after the second product, not beside it (registers)
  int fl = 0, fln = 2, buf = 0;
  int t = advance(fl), tn = -1;
  float st[32];                                        // tile t's scores
  float mx;
  typename Score<MODE>::At at[2];
  auto places = [&](const int t) __attribute__((always_inline)) {
    at[0] = sc.template at<true>(t * MA_KT + 4 * lhi - pos);
    at[1] = sc.template at<true>(t * MA_KT + 32 + 4 * lhi - pos);
    mx = -MA_INF;
  };
  auto finish = [&](auto e_, const f32x16 (&acc)[2]) __attribute__((always_inline)) {
    constexpr int e = decltype(e_)::value;
    st[e] = sc.score(acc[e >> 4][e & 15], at[e >> 4], ma_row(e & 15));
    mx = fmaxf(mx, st[e]);
  };
  // masks tile t's scores (document numbers in buffer `buf`)
  auto mask = [&](const int t, const int buf) __attribute__((always_inline)) {
    mx = -MA_INF;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      if (docs) ma_mask<true>(st + k2 * 16, t * MA_KT + k2 * 32, lhi, lim, sdoc + buf * MA_KT + k2 * 32, dq);
      else ma_mask<false>(st + k2 * 16, t * MA_KT + k2 * 32, lhi, lim, nullptr, 0);
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) mx = fmaxf(mx, st[e]);
  };
  if (t >= 0) {
    load_k(t, 0, fl);
    tn = advance(fln);
    if (tn >= 0) load_k(tn, 1, fln);
    load_v(t, 0, fl);
    ma_dma_wait();
    __syncthreads();
    f32x16 acc[2] = {ma_zero(), ma_zero()};
    ma_stream<NP, 4, v8>([&](auto x) { return TL::template row_frag<v8>(smem, kbase, (x & 1) * 32, x >> 1); },
                         [&](auto x, const v8 kf) { acc[x & 1] = ma_mfma(kf, qf[x >> 1], acc[x & 1]); });
    places(t);
    ma_each<0, 32>([&](auto e) __attribute__((always_inline)) { finish(e, acc); });
    if (!(fl & 2)) mask(t, 0);
    rs.rise(mx);
  }
  // one tile: its probabilities beside the products of the next tile's scores, then its second product beside the next scores' cap, bias and
  // maximum.  Each product is followed by the arithmetic of EPP scores, in this order, so that the matrix pipe and the vector pipe work on
  // one wave at the same time.
  ma_loads_landed();
  while (t >= 0) {
    ma_dma_wait();
    __syncthreads();                                   // the next K and this V have landed everywhere, and everyone is done with the other buffers
    int flnn = 2, tnn = -1;
    if (tn >= 0) {
      load_v(tn, buf ^ 1, fln);
      tnn = advance(flnn);
      if (tnn >= 0) load_k(tnn, buf, flnn);
    }
    const float base = rs.base();
    v8 pf[4];
    float l0 = 0.f, l1 = 0.f;
    auto probs = [&](auto x) __attribute__((always_inline)) {
      ma_each<0, EPP>([&](auto y) __attribute__((always_inline)) {
        constexpr int e = decltype(x)::value * EPP + decltype(y)::value;
        const float pr = __builtin_amdgcn_exp2f(st[e] - base);
        if (e & 1) l1 += pr; else l0 += pr;
        pf[e >> 3][e & 7] = (T)pr;                     // rounded to nearest: maskattn.h, ma_pack
      });
    };
    const char* const sk = smem + (buf ^ 1) * TBYTES;
    const char* const sv = smem + (2 + buf) * TBYTES;
    const int kb = D == 64 || LATE ? ma_opaque(kbase) : kbase, vb = D == 64 || LATE ? ma_opaque(vbase) : vbase;      // (D = 64 has 168 registers: the swizzled addresses are made per tile)
    f32x16 acc[2] = {ma_zero(), ma_zero()};
    // (after the last tile the scores are those of an old buffer and nobody looks at them: a branch here would move the exponentials in front of it)
    ma_stream<NP, 4, v8>([&](auto x) { return TL::template row_frag<v8>(sk, kb, (x & 1) * 32, x >> 1); },
                         [&](auto x, const v8 kf) { acc[x & 1] = ma_mfma(kf, qf[x >> 1], acc[x & 1]); probs(x); });
    rs.l += l0 + l1;
    places(tn);
    ma_stream<NP, 4, v8>([&](auto x) { return TL::template tr_frag<v8>(sv, vb, x % DT, x / DT * 16); },
                         [&](auto x, const v8 vf) {
                           rs.o[x % DT] = ma_mfma(vf, pf[x / DT], rs.o[x % DT]);
                           if constexpr (!LATE)
                             ma_each<0, EPP>([&](auto y) __attribute__((always_inline)) { finish(MaIdx<decltype(x)::value * EPP + decltype(y)::value>{}, acc); });
                         });
    if constexpr (LATE) ma_each<0, 32>([&](auto e) __attribute__((always_inline)) { finish(e, acc); });
    if (tn >= 0) {
      if (!(fln & 2)) mask(tn, buf ^ 1);
      rs.rise(mx);
    }
    buf ^= 1;
    t = tn; fl = fln;
    tn = tnn; fln = flnn;
  }

  // ---- epilogue: O[i][d] = O^T[d][i] / l
  const MgldMaskAttn& pe = D == 128 ? ma_late_args() : p;
  const float l = rs.l + __shfl_xor(rs.l, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float z = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) z += rs.o[dt][r] * 0.f;
  // an infinity or NaN came in, perhaps of a value that the row does not see.  (Where the sum of the probabilities is not finite, a score that it sees was not: all NaN.)
  const unsigned long long bz = __ballot(z != z && l - l == 0.f);
  unsigned bad = (unsigned)bz | (unsigned)(bz >> 32);
  if (i < pe.Nq) {
    if (pe.lse && lhi == 0) pe.lse[((int64_t)b * pe.heads + h) * pe.Nq + i] = l == 0.f ? -MA_INF : (rs.unit() + __builtin_amdgcn_logf(l)) * MA_LN2;
    T* const o = (T*)pe.O + b * pe.o_sb + (int64_t)i * pe.o_si + h * pe.o_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int d = dt * 32 + rg * 8 + lhi * 4;
        typedef T t4 __attribute__((ext_vector_type(4)));
        if (d < pe.head_dim)
          *(t4*)(o + d) = t4{(T)(rs.o[dt][rg * 4] * inv), (T)(rs.o[dt][rg * 4 + 1] * inv), (T)(rs.o[dt][rg * 4 + 2] * inv), (T)(rs.o[dt][rg * 4 + 3] * inv)};
      }
  }
  while (bad) {
    const int r = __builtin_ctz(bad);
    bad &= bad - 1;
    if (iw + r < pe.Nq) ma_slow_row<T>(D == 128 ? ma_late_args() : p, b, h, iw + r);
  }
}

// ---- few rows over many keys ----------------------------------------------------------------------------------------------------------
// Rows of the query heads that share a key head are packed: packed row r = (query i = r / G, head of the group g = r % G); a block takes 32 of
// them and one slice of the tiles, its 4 waves every fourth tile each, by DMA into LDS of their own (no barrier in the loop).  The waves' states
// meet in LDS, the slices' in ma_join_kernel through fp32 partial results in the work buffer.
template <typename T, int D, int MODE>
__global__ __launch_bounds__(256, 2) void ma_split_kernel(const MgldMaskAttn p, const i32x4* __restrict__ kdoc, const int nsplit, const int nrb, float* part) {
  typedef typename MaVec<T>::v8 v8;
  typedef Tile<D> TL;
  constexpr int DK = D / 16, DT = D / 32, KH = 32;
  constexpr int TBYTES = KH * TL::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];              // per wave [2] x {K, V} of 32 keys (later: its O [32][D] fp32), doc numbers, m / l, distance rows
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lhi = lane >> 5;
  int* const sdoc = (int*)(smem + 16 * TBYTES) + wave * 2 * MA_KT;         // (a DMA writes 64 words)
  float* const sml = (float*)(smem + 16 * TBYTES) + 8 * MA_KT;             // [4][2][32]
  float* const srel = sml + 256;
  const int G = p.heads / p.kv_heads, rows = G * p.Nq;
  const int split = blockIdx.x, hk = blockIdx.y % p.kv_heads, rb = blockIdx.y / p.kv_heads, b = blockIdx.z;
  const BatchSpan bs(p, b);
  const bool docs = p.doc_q != nullptr;
  const int ntk = (p.Nkv + MA_KT - 1) / MA_KT;
  if (docs) kdoc += (int64_t)b * ntk;

  const int r = rb * 32 + l31;
  const bool rok = r < rows;
  const int i = rok ? r / G : 0, h = hk * G + (rok ? r % G : 0), pos = bs.pos0 + i;
  const int dq = docs && rok ? p.doc_q[b * p.doc_q_sb + i] : -1;
  const int lim = rok && (!docs || dq >= 0) ? bs.limit(p, pos) : 0;              // (0 where a row has no document)
  const int if_ = rb * 32 / G, il = (min(rb * 32 + 32, rows) - 1) / G;     // queries of this block
  const RowGroup g = ma_row_group(p, bs, b, if_, il - if_ + 1);
  const T* __restrict__ Kp = (const T*)p.K + b * p.k_sb + hk * p.k_sh;
  const T* __restrict__ Vp = (const T*)p.V + b * p.v_sb + hk * p.v_sh;
  const int d8 = p.head_dim / 8;
  v8 zero;
#pragma unroll
  for (int e = 0; e < 8; ++e) zero[e] = (T)0.f;
  v8 qf[DK];
  {
    const T* q = (const T*)p.Q + b * p.q_sb + (int64_t)i * p.q_si + h * p.q_sh;
#pragma unroll
    for (int ks = 0; ks < DK; ++ks) qf[ks] = rok && ks * 2 + lhi < d8 ? *(const v8*)(q + ks * 16 + lhi * 8) : zero;
  }
  // a lane's head differs from its neighbour's: the distance rows of the group's heads lie side by side
  if (MODE & MA_REL) ma_load_rel(p, hk * G, G, srel);
  __syncthreads();
  const Score<MODE> sc(p, h, srel + (rok ? r % G : 0) * ma_rel_floats(p.reach));

  // this block's tiles: an equal share of those below the rows' limits
  const int nt = ma_tiles(g.lim_max), share = (nt + nsplit - 1) / nsplit;
  const int ta = min(split * share, nt), tb = min(ta + share, nt);
  int w0 = ta - 64;
  unsigned long long act = 0, full = 0;
  int cur = -1, half = 1, curfull = 0;
  auto advance = [&](int& fullf) __attribute__((always_inline)) {      // next 32-key half tile, or -1
    if (half == 0 && (cur * 2 + 1) * KH < g.lim_max) { half = 1; fullf = curfull; return cur * 2 + 1; }
    while (!act) {
      w0 += 64;
      if (w0 >= tb) return -1;
      const int t = w0 + lane;
      const i32x4 dt = docs && t < ntk ? kdoc[t] : i32x4{0x7fffffff, -1, 0, 0};
      ma_window(p, g, dt, t, act, full);
      act &= __ballot(t < tb && ((t - ta) & 3) == wave);
    }
    const int c = __builtin_ctzll(act);
    act &= act - 1;
    cur = __builtin_amdgcn_readfirstlane(w0 + c); half = 0; curfull = (int)((full >> c) & 1);
    fullf = curfull;
    return cur * 2;
  };

  const TileDma<D, KH, 1> dk(0, lane, p.k_si, p.head_dim), dv(0, lane, p.v_si, p.head_dim);
  const unsigned lds0 = ma_lds_addr(smem) + __builtin_amdgcn_readfirstlane(wave) * 4 * TBYTES;
  const unsigned lds_doc = ma_lds_addr(smem) + 16 * TBYTES + __builtin_amdgcn_readfirstlane(wave) * 2 * MA_KT * 4;
  auto load_half = [&](const int t, const int buf) __attribute__((always_inline)) {
    const int k0 = t * KH;
    const unsigned a = lds0 + buf * 2 * TBYTES;
    dk.load(Kp, (int64_t)k0 * p.k_si * 2, p.k_si, g.lim_max - k0, a);
    dv.load(Vp, (int64_t)k0 * p.v_si * 2, p.v_si, g.lim_max - k0, a + TBYTES);
    if (docs) ma_dma4(lds_doc + buf * MA_KT * 4, lane, min(KH, g.lim_max - k0), p.doc_k + b * p.doc_k_sb + k0);
  };
  RowState<T, DT> rs;
  const int kbase = TL::row_base(lane), vbase = TL::tr_base(lane);
  int fl = 0, buf = 0;
  int t = advance(fl);
  if (t >= 0) load_half(t, 0);
  while (t >= 0) {
    ma_dma_wait();                                       // the wave's own tile: no other wave reads it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int fln = 0;
    const int tn = advance(fln);
    if (tn >= 0) load_half(tn, buf ^ 1);
    const char* const sk = smem + wave * 4 * TBYTES + buf * 2 * TBYTES;
    const char* const sv = sk + TBYTES;
    __builtin_amdgcn_sched_barrier(0);
    f32x16 acc = ma_zero();
    ma_stream<DK, 4, v8>([&](auto x) { return TL::template row_frag<v8>(sk, kbase, 0, x); }, [&](auto x, const v8 kf) { acc = ma_mfma(kf, qf[x], acc); });
    const int k0 = t * KH;
    const auto at = sc.template at<true>(k0 + 4 * lhi - pos);
    float st[16], mx = -MA_INF;
#pragma unroll
    for (int e = 0; e < 16; ++e) st[e] = sc.score(acc[e], at, ma_row(e));
    if (!fl) {
      if (docs) ma_mask<true>(st, k0, lhi, lim, sdoc + buf * MA_KT, dq);
      else ma_mask<false>(st, k0, lhi, lim, nullptr, 0);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, st[e]);
    rs.rise(mx);
    const float base = rs.base();
    v8 pf[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      st[e] = __builtin_amdgcn_exp2f(st[e] - base);
      rs.l += st[e];
    }
    pf[0] = ma_pack<T>(st);
    pf[1] = ma_pack<T>(st + 8);
    ma_stream<2 * DT, 4, v8>([&](auto x) { return TL::template tr_frag<v8>(sv, vbase, x % DT, x / DT * 16); },
                             [&](auto x, const v8 vf) { rs.o[x % DT] = ma_mfma(vf, pf[x / DT], rs.o[x % DT]); });
    t = tn; fl = fln; buf ^= 1;
  }

  // ---- the four waves' states meet: o * 2^(m_w - M)
  const float l = rs.l + __shfl_xor(rs.l, 32, 64);
  __syncthreads();                                       // every wave is done with its tiles
  if (lhi == 0) { sml[wave * 64 + l31] = rs.unit(); sml[wave * 64 + 32 + l31] = l; }
  float* const so = (float*)smem + wave * 32 * D;        // [32 rows][D] fp32 = the wave's two tiles' bytes
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg)
      *(f32x4*)(so + l31 * D + ((dt * 32 + rg * 8 + lhi * 4) ^ ((l31 & 7) * 4))) =
          f32x4{rs.o[dt][rg * 4], rs.o[dt][rg * 4 + 1], rs.o[dt][rg * 4 + 2], rs.o[dt][rg * 4 + 3]};
  __syncthreads();
  for (int rr = wave; rr < 32; rr += 4) {                // a wave per row, lanes over d
    const int pr = rb * 32 + rr;
    if (pr >= rows) break;
    float M = -MA_INF;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w * 64 + rr]);
    float L = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = sml[w * 64 + rr];
      const float f = mw == -MA_INF ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      L += sml[w * 64 + 32 + rr] * f;
      const float* ow = (const float*)smem + w * 32 * D + rr * D;
      a0 += ow[lane ^ ((rr & 7) * 4)] * f;
      if (D == 128) a1 += ow[(lane + 64) ^ ((rr & 7) * 4)] * f;
    }
    const int ii = pr / G, hh = hk * G + pr % G;
    if (nsplit > 1) {
      const int64_t slot = (((int64_t)b * p.heads + hh) * p.Nq + ii) * nsplit + split;
      float* const po = part + slot * (D + 2);
      po[lane] = a0;
      if (D == 128) po[lane + 64] = a1;
      if (lane == 0) { po[D] = M; po[D + 1] = L; }           // the maximum in log2 units
    } else {
      const bool bad = L - L == 0.f && __any(a0 * 0.f != a0 * 0.f || a1 * 0.f != a1 * 0.f);      // (L not finite: a visible score was not, all NaN)
      if (p.lse && lane == 0) p.lse[((int64_t)b * p.heads + hh) * p.Nq + ii] = L == 0.f ? -MA_INF : (M + __builtin_amdgcn_logf(L)) * MA_LN2;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      T* const o = (T*)p.O + b * p.o_sb + (int64_t)ii * p.o_si + hh * p.o_sh;
      if (lane < p.head_dim) o[lane] = (T)(a0 * inv);
      if (lane + 64 < p.head_dim) o[lane + 64] = (T)(a1 * inv);
      if (bad) ma_slow_row<T>(p, b, hh, ii);
    }
  }
}

// joins the slices of one row: a wave per row
template <typename T, int D>
__global__ __launch_bounds__(64) void ma_join_kernel(const MgldMaskAttn p, const float* part, const int nsplit) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const float* const po = part + row * nsplit * (D + 2);
  float M = -MA_INF;
  for (int s = lane; s < nsplit; s += 64) M = fmaxf(M, po[(int64_t)s * (D + 2) + D]);
  M = wave_max(M);
  float L = 0.f, a0 = 0.f, a1 = 0.f;
  for (int s = 0; s < nsplit; ++s) {
    const float* const ps = po + (int64_t)s * (D + 2);
    const float f = ps[D] == -MA_INF ? 0.f : __builtin_amdgcn_exp2f(ps[D] - M);
    L += ps[D + 1] * f;
    a0 += ps[lane] * f;
    if (D == 128) a1 += ps[lane + 64] * f;
  }
  const int i = (int)(row % p.Nq), h = (int)(row / p.Nq % p.heads), b = (int)(row / p.Nq / p.heads);
  if (p.lse && lane == 0) p.lse[row] = L == 0.f ? -MA_INF : (M + __builtin_amdgcn_logf(L)) * MA_LN2;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* const o = (T*)p.O + b * p.o_sb + (int64_t)i * p.o_si + h * p.o_sh;
  if (lane < p.head_dim) o[lane] = (T)(a0 * inv);
  if (lane + 64 < p.head_dim) o[lane + 64] = (T)(a1 * inv);
  if (L - L == 0.f && __any(a0 * 0.f != a0 * 0.f || a1 * 0.f != a1 * 0.f)) ma_slow_row<T>(p, b, h, i);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
struct Plan { bool split; int nsplit, nrb; };
// few rows: when one block per 128 rows would leave most of the card idle and there are keys to share out.  Row blocks | split, us (fp16, causal):
//   32 / 8 heads of 128, 512 keys: 16 rows 20.1 | 13.4, 17 rows 20.0 | 13.5, 128 rows 19.4 | 16.4;  16 sequences of 2048 keys: 16 rows 99 | 55, 17 rows 106 | 75
//   (from 17 rows on these count as many rows, and lose a third);  16 heads of 64, 4096 keys: 17 rows 109 | 17, 128 rows 90 | 21, 512 rows 88 | 35;
//   4 heads of 128, 4096 keys: 512 rows 114 | 34, 2048 rows 114 | 60;  16 heads of 64, 77 keys: 8 rows 7.3 | 7.0, 16 rows 7.3 | 8.4;  2 heads of 64, 300 rows: 960 keys 25.5 | 12.4
//   (row blocks: fewer than 16 tiles), 1024 keys 27.2 | 12.5.  Both borders are on the safe side of the crossing, not at it.
Plan ma_plan(const MgldMaskAttn* p) {
  Plan pl{false, 1, 1};
  const int G = p->heads / p->kv_heads, nt = ma_tiles(p->Nkv);
  const int64_t rows = (int64_t)G * p->Nq;
  const int64_t blocks = (int64_t)p->batch * p->heads * ((p->Nq + 127) / 128);
  const int64_t packed = (int64_t)p->batch * p->kv_heads * ((rows + 31) / 32);
  const bool rel_fits = !p->rel || (int64_t)G * ma_rel_floats(p->reach) * 4 <= 28 * 1024;       // (beside 131 KB of tiles)
  pl.split = rel_fits && (rows + 31) / 32 * p->kv_heads <= 65535 && p->batch <= 65535 && (p->Nq <= 16 || (blocks * 4 <= 256 && nt >= 16));
  if (!pl.split) return pl;
  pl.nrb = (int)((rows + 31) / 32);
  // two blocks per CU; a slice keeps at least one tile for each of its four waves
  int64_t n = (2 * 256 + packed - 1) / packed;
  if (n > (nt + 3) / 4) n = (nt + 3) / 4;
  if (n > 128) n = 128;
  pl.nsplit = n < 1 ? 1 : (int)n;
  return pl;
}

template <typename T, int D, int MODE>
int ma_launch(const MgldMaskAttn& p, hipStream_t st) {
  const Plan pl = ma_plan(&p);
  const i32x4* kdoc = (const i32x4*)p.work;
  float* part = (float*)((char*)p.work + ma_doc_bytes(&p));
  const int nrel = p.rel ? ma_rel_floats(p.reach) : 0;
  if (p.doc_q) {
    const int rc = ma_doc_tiles(p, p.work, st);
    if (rc) return rc;
  }
  if (!pl.split) {
    const int64_t nqb = (p.Nq + 127) / 128, nb = nqb * p.batch * p.heads;
    MGLD_REQUIRE(nb <= 0x7fffffff, "masked_attention: grid");
    const int lds = 4 * MA_KT * Tile<D>::RB + 2 * MA_KT * 4 + nrel * 4;
    static_assert(4 * MA_KT * Tile<D>::RB + 2 * MA_KT * 4 + (2 * MA_MAX_REACH + 1 + 2 * MA_PAD) * 4 <= 80 * 1024, "two blocks per CU");
    if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)ma_fwd_kernel<T, D, MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    ma_fwd_kernel<T, D, MODE><<<dim3((unsigned)nb), 256, lds, st>>>(p, kdoc, (int)nqb);
    return mgld_check_launch("masked_attention");
  }
  const int G = p.heads / p.kv_heads;
  const int lds = 16 * 32 * Tile<D>::RB + 8 * MA_KT * 4 + 256 * 4 + G * nrel * 4;
  if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)ma_split_kernel<T, D, MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  ma_split_kernel<T, D, MODE><<<dim3(pl.nsplit, pl.nrb * p.kv_heads, p.batch), 256, lds, st>>>(p, kdoc, pl.nsplit, pl.nrb, part);
  if (pl.nsplit > 1) ma_join_kernel<T, D><<<dim3((unsigned)((int64_t)p.batch * p.heads * p.Nq)), 64, 0, st>>>(p, part, pl.nsplit);
  return mgld_check_launch("masked_attention");
}
bool ma_aligned(const void* ptr, const int64_t sb, const int64_t si, const int64_t sh) {
  return ptr && (uintptr_t)ptr % 16 == 0 && sb % 8 == 0 && si % 8 == 0 && sh % 8 == 0;
}

}  // namespace

int ma_check(const MgldMaskAttn* p, const bool grad) {
  MGLD_REQUIRE(p && p->batch >= 0 && p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0, "masked_attention: heads must be a multiple of kv_heads");
  MGLD_REQUIRE(p->Nq >= 0 && p->Nkv >= 0 && p->Nq <= (1 << 30) && p->Nkv <= (1 << 30), "masked_attention: lengths");
  MGLD_REQUIRE(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "masked_attention: head_dim must be a multiple of 8 up to 128");
  MGLD_REQUIRE(p->scale > 0.f && p->scale < 3e38f && p->softcap >= 0.f && p->softcap < 3e38f, "masked_attention: scale > 0, softcap >= 0");
  MGLD_REQUIRE(p->q_pos0 >= -(1 << 30) && p->q_pos0 <= (1 << 30) , "masked_attention: q_pos0");
  MGLD_REQUIRE(!p->rel || (p->reach >= 0 && p->reach <= MA_MAX_REACH), "masked_attention: reach up to 1024");
  MGLD_REQUIRE(!p->rel || !p->slopes, "masked_attention: slopes or rel, not both");
  MGLD_REQUIRE(!grad || !p->rel || (int64_t)(p->heads / p->kv_heads) * ma_rel_floats(p->reach) * 4 <= 92 * 1024,
               "masked_attention_grad: the distance rows of the query heads that share a key head must fit 92 KB");
  MGLD_REQUIRE(!p->prefix || p->causal, "masked_attention: prefix needs causal");
  MGLD_REQUIRE((p->doc_q != nullptr) == (p->doc_k != nullptr) || p->Nq == 0 || p->Nkv == 0, "masked_attention: doc_q and doc_k go together");
  if (p->batch == 0 || (p->Nq == 0 && !grad)) return MGLD_OK;
  if (p->Nq > 0) {
    MGLD_REQUIRE(ma_aligned(p->Q, p->q_sb, p->q_si, p->q_sh) && (grad || ma_aligned(p->O, p->o_sb, p->o_si, p->o_sh)), "masked_attention: q / o must be 16-byte aligned with strides of multiples of 8");
    if (grad) MGLD_REQUIRE(ma_aligned(p->dO, p->do_sb, p->do_si, p->do_sh) && ma_aligned(p->dQ, p->dq_sb, p->dq_si, p->dq_sh) && p->lse, "masked_attention_grad: do / dq alignment, lse");
  }
  // a tile's rows are addressed with 31-bit byte offsets (its base with 64 bits)
  auto row_ok = [](const int64_t si) { return si >= 0 && si < (1 << 23); };
  MGLD_REQUIRE(row_ok(p->q_si) && row_ok(p->k_si) && row_ok(p->v_si) && (!grad || row_ok(p->do_si)), "masked_attention: row strides must be below 2^23 elements");
  if (p->Nkv > 0) {
    MGLD_REQUIRE(ma_aligned(p->K, p->k_sb, p->k_si, p->k_sh) && ma_aligned(p->V, p->v_sb, p->v_si, p->v_sh), "masked_attention: k / v must be 16-byte aligned with strides of multiples of 8");
    if (grad) MGLD_REQUIRE(ma_aligned(p->dK, p->dk_sb, p->dk_si, p->dk_sh) && ma_aligned(p->dV, p->dv_sb, p->dv_si, p->dv_sh), "masked_attention_grad: dk / dv alignment");
  }
  return MGLD_OK;
}

int ma_doc_tiles(const MgldMaskAttn& p, void* out, hipStream_t st) {
  MGLD_REQUIRE(p.batch <= 65535, "masked_attention: batch with documents up to 65535");
  const int n = ma_tiles(p.Nkv) + ma_tiles(p.Nq);
  if (n > 0) ma_doc_tiles_kernel<<<dim3(n, p.batch), 64, 0, st>>>(p.doc_k, p.doc_q, p.doc_k_sb, p.doc_q_sb, p.Nkv, p.Nq, p.batch, (i32x4*)out);
  return mgld_check_launch("masked_attention documents");
}

extern "C" int64_t mgld_masked_attention_work(const MgldMaskAttn* p) {
  if (!p || ma_check(p, false) || p->batch == 0 || p->Nq == 0) return 0;
  const Plan pl = ma_plan(p);
  const int D = p->head_dim <= 64 ? 64 : 128;
  return ma_doc_bytes(p) + (pl.nsplit > 1 ? (int64_t)p->batch * p->heads * p->Nq * pl.nsplit * (D + 2) * 4 : 0);
}

extern "C" int mgld_masked_attention(const MgldMaskAttn* p, void* stream) {
  const int rc = ma_check(p, false);
  if (rc || p->batch == 0 || p->Nq == 0) return rc;
  const int64_t need = mgld_masked_attention_work(p);
  MGLD_REQUIRE(need == 0 || (p->work && (uintptr_t)p->work % 16 == 0 && p->work_bytes >= need), "masked_attention: work buffer too small");
  hipStream_t st = (hipStream_t)stream;
  MA_DISPATCH(ma_launch, p, st)
}
