// maskattn_grad.hip — gradient of the masked attention (maskattn.hip) from its output and log-sum-exp.
//
//   P = exp(s - lse),  dP = dO V^T,  D = rowsum(P dP) = dO . o,  dS = P (dP - D),  dT = dS (1 - (u / softcap)^2)
//   dV = P^T dO,  dQ = scale dT K,  dK = scale dT^T Q,  dRel[h][c] = sum of dS over the pairs at distance c
//
// Passes over the visible pairs that recompute the scores, so that every sum has one owner and a fixed order (no atomics; 9 products
// instead of 5):
//  * ma_dq_kernel, per 128 query rows, goes over the keys twice: D = sum P dP first (from the rounded o, D would be off by 2^-9 sum |do o| in bf16, which
//    the sums over rows keep: dRel lost three digits), then S^T = K Q^T and dP^T = V dO^T again (a lane holds keys of ONE query row) and
//    dQ^T += K^T dT^T; K read both ways from one LDS tile.  With a relative bias it also adds dS along the diagonals: a 32 x 32 block goes through LDS, lane c sums diagonal c;
//    blocks wholly beyond the reach only add to the two end sums.
//  * ma_dkv_kernel, per 128 keys of a key head: S = Q K^T and dP = dO V^T (a lane holds query rows of ONE key), dV^T += dO^T P, dK^T += Q^T dT over
//    all query heads of the group.  Where that gives too few blocks, the (head, tile) list is dealt to `nsp` blocks whose fp32 sums are added.
// Bounds and figures: 2 x 2048 tokens, 16 / 4 heads of 128, causal with a prefix: dQ 157 us, dK / dV 148 + 13 us (forward 66).  At d = 128 the LDS reads of 32 rows or keys
// per wave take as long as the products (wider waves need more registers than there are), and two waves per SIMD hide little of the scores'
// arithmetic behind them.  With a learned bias (4 x 1024 tokens, 16 heads of 64): dQ 103 us, dK / dV 84 us (forward 40): the diagonals pass through LDS.
// fp16 operands have 5 exponent bits: dT is scaled by powers of two before its rounding, per row in ma_dq, by one number for the call in ma_dkv.  The scale
// comes from dS itself: |dS| = P |dP - D| <= max(P |dP|) + |D|, which the pass for D has at hand (one more maximum per score), so that bound goes to
// 2^13 .. 2^14 whatever the sizes of dO and V: nothing overflows, and what is rounded to a subnormal lies 2^27 below the largest.  P is rounded as 2^10 P there.
// bf16 has the exponents and needs none of it.
#include "maskattn.h"

namespace {

constexpr int MA_DS_EXP = 13;          // fp16: the largest |dS| a row or a call can have goes to [2^13, 2^14)

// the largest finite bound of |dS| -> out[0]
__global__ __launch_bounds__(1024) void ma_amax_kernel(const float* amax, const int64_t rows, float* out) {
  __shared__ float sm[16];
  float m = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    const float a = amax[i];
    if (a < MA_INF) m = fmaxf(m, a);
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) m = fmaxf(m, sm[w]);
    out[0] = m;
  }
}
// the power of two that brings amax into [2^e, 2^(e+1)); 1 where amax is 0 or not finite
__device__ __forceinline__ float ma_pow2_to(const float amax, const int e) {
  if (!(amax > 0.f && amax < MA_INF)) return 1.f;
  const int k = e + 127 - (int)(__float_as_uint(amax) >> 23);            // amax = f 2^(x - 127): the factor is 2^(e - x + 127)
  return __uint_as_float((unsigned)(min(max(k, -126), 127) + 127) << 23);
}

struct GradWork {
  float *delta, *amax, *gmax, *rel, *kv;
  const i32x4* doc;
};

// ---- dQ (and dRel) ------------------------------------------------------------------------------------------------------------------------
template <typename T, int D, int MODE, bool REL>
__global__ __launch_bounds__(256, 2) void ma_dq_kernel(const MgldMaskAttn p, const GradWork w, const int nqb) {
  static_assert(!REL || (MODE & MA_REL), "the distance row's gradient");
  typedef typename MaVec<T>::v8 v8;
  typedef Tile<D> TL;
  constexpr int DK = D / 16, DT = D / 32;
  constexpr int TBYTES = MA_KT * TL::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2] x {K, V}, doc numbers [2][64], the distance row, REL: per wave block [32][33] and sums
  int* const sdoc = (int*)(smem + 4 * TBYTES);
  float* const srel = (float*)(sdoc + 2 * MA_KT);
  const int nrel = 2 * p.reach + 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lhi = lane >> 5;
  const int nbh = p.batch * p.heads;
  int bh, qb;
  if (nbh % 8 == 0) {            // (block order: maskattn.hip)
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
  const int ntk = ma_tiles(p.Nkv);
  const i32x4* const kdoc = w.doc + (int64_t)b * ntk;
  const T* __restrict__ Kp = (const T*)p.K + b * p.k_sb + hk * p.k_sh;
  const T* __restrict__ Vp = (const T*)p.V + b * p.v_sb + hk * p.v_sh;
  const int d8 = p.head_dim / 8;
  v8 zero;
#pragma unroll
  for (int e = 0; e < 8; ++e) zero[e] = (T)0.f;
  const int i = iw + l31, pos = bs.pos0 + i;
  const bool rok = i < p.Nq;
  const int dq = docs && rok ? p.doc_q[b * p.doc_q_sb + i] : -1;
  const int lim = rok && (!docs || dq >= 0) ? bs.limit(p, pos) : 0;              // (0 where a row has no document)
  const int64_t srow = ((int64_t)b * p.heads + h) * p.Nq + i;
  const float lse = rok ? p.lse[srow] : -MA_INF;
  const float lse2 = lse == -MA_INF ? MA_INF : lse * MA_LOG2E;          // a row that sees nothing: P = 0
  v8 qf[DK], gf[DK];
#pragma unroll
  for (int ks = 0; ks < DK; ++ks) {
    const bool ok = rok && lse2 < MA_INF && ks * 2 + lhi < d8;         // a row that sees nothing adds nothing, whatever it holds
    qf[ks] = ok ? *(const v8*)((const T*)p.Q + b * p.q_sb + (int64_t)i * p.q_si + h * p.q_sh + ks * 16 + lhi * 8) : zero;
    gf[ks] = ok ? *(const v8*)((const T*)p.dO + b * p.do_sb + (int64_t)i * p.do_si + h * p.do_sh + ks * 16 + lhi * 8) : zero;
  }
  constexpr bool F16 = __is_same(T, f16);
  if (MODE & MA_REL) ma_load_rel(p, h, 1, srel);
  float* const sblk = srel + ((MODE & MA_REL) ? ma_rel_floats(p.reach) : 0) + wave * (32 * 33 + nrel);
  float* const sacc = sblk + 32 * 33;
  if (REL)
    for (int e = lane; e < nrel; e += 64) sacc[e] = 0.f;
  float far_l = 0.f, far_r = 0.f;
  const Score<MODE> sc(p, h, srel);

  const int nt = ma_tiles(gb.lim_max);
  int w0 = -64;
  unsigned long long bact = 0, wact = 0, wfull = 0, bfull = 0, pads = 0;
  auto advance = [&](int& flags) __attribute__((always_inline)) {
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
    return __builtin_amdgcn_readfirstlane(w0 + c);
  };
  const TileDma<D, MA_KT, 4> dk(wave, lane, p.k_si, p.head_dim), dv(wave, lane, p.v_si, p.head_dim);
  const unsigned lds0 = ma_lds_addr(smem);
  auto load_tile = [&](const int t, const int buf, const int flags) __attribute__((always_inline)) {
    const int k0 = t * MA_KT;
    const unsigned a = lds0 + buf * 2 * TBYTES;
    const int32_t* const ids = docs ? p.doc_k + b * p.doc_k_sb + k0 : nullptr;
    dk.load(Kp, (int64_t)k0 * p.k_si * 2, p.k_si, gb.lim_max - k0, a, flags & 4, [&](const int r) { return ids[r] < 0; });       // (keys no row of the block sees hold anything)
    dv.load(Vp, (int64_t)k0 * p.v_si * 2, p.v_si, gb.lim_max - k0, a + TBYTES, flags & 4, [&](const int r) { return ids[r] < 0; });
    if (docs && wave == 0) ma_dma4(lds0 + 4 * TBYTES + buf * MA_KT * 4, lane, bs.len - k0, ids);
  };

  const int kbase = TL::row_base(lane), tbase = TL::tr_base(lane);
  // a 32-key half of tile t: scores and dP
  auto products = [&](const char* sk, const char* sv, const int k2, f32x16& s, f32x16& dp) __attribute__((always_inline)) {
    s = ma_zero();
    dp = ma_zero();
    const int kb = REL && D == 128 && (MODE & MA_WIDE) ? ma_opaque(kbase) : kbase;       // (registers: the swizzled addresses are made per half)
    ma_stream<2 * DK, REL && D == 128 ? 3 : 4, v8>([&](auto x) { return TL::template row_frag<v8>(x & 1 ? sv : sk, kb, k2 * 32, x >> 1); },
                             [&](auto x, const v8 f) { if (x & 1) dp = ma_mfma(f, gf[x >> 1], dp); else s = ma_mfma(f, qf[x >> 1], s); });
  };
  int buf = 0;
  float delta = 0.f, top = 0.f;
  {                                                    // D = sum P dP; fp16: top = max P |dP|
    int fl = 0, fln = 0;
    int t = advance(fl);
    if (t >= 0) load_tile(t, buf, fl);
    ma_loads_landed();
    while (t >= 0) {
      ma_dma_wait();
      __syncthreads();
      const int tn = advance(fln);
      if (tn >= 0) load_tile(tn, buf ^ 1, fln);
      if (fl & 1) {
        const char* const sk = smem + buf * 2 * TBYTES;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          f32x16 s, dp;
          products(sk, sk + TBYTES, k2, s, dp);
          const int k0 = t * MA_KT + k2 * 32;
          const auto at = sc.template at<true>(k0 + lhi * 4 - pos);
        const int ll = ma_opaque(lim - (k0 + lhi * 4));
#pragma unroll
          for (int rg = 0; rg < 4; ++rg) {
            i32x4 dk4 = {dq, dq, dq, dq};
            if (docs && !(fl & 2)) dk4 = *(const i32x4*)(sdoc + buf * MA_KT + k2 * 32 + rg * 8 + lhi * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = rg * 4 + e;
              float sq = 0.f;
              float x = sc.template prob<true>(s[r], at, rg * 8 + e, lse2, sq) * dp[r];
              if (!(fl & 2)) x = (rg * 8 + e < ll) & (dk4[e] == dq) ? x : 0.f;
              delta += x;
              if (F16) top = fmaxf(top, fabsf(x));
            }
          }
        }
      }
      buf ^= 1;
      t = tn; fl = fln;
    }
    delta += __shfl_xor(delta, 32, 64);
    if (rok && lhi == 0) w.delta[srow] = delta;
    if (F16) {
      top = fmaxf(top, __shfl_xor(top, 32, 64)) + fabsf(delta);
      const float am = wave_max(top < MA_INF ? top : 0.f);
      if (lane == 0) w.amax[(int64_t)blockIdx.x * 4 + wave] = am;
    }
    __syncthreads();                                   // everyone is done with both buffers
    w0 = -64;
    bact = 0;
  }

  const float up = F16 ? ma_pow2_to(top, MA_DS_EXP) : 1.f;             // fp16: dT is rounded as dT * up
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = ma_zero();
  int fl = 0, fln = 0;
  int t = advance(fl);
  if (t >= 0) load_tile(t, buf, fl);
  ma_loads_landed();
  while (t >= 0) {
    ma_dma_wait();
    __syncthreads();
    const int tn = advance(fln);
    if (tn >= 0) load_tile(tn, buf ^ 1, fln);
    if (fl & 1) {
      const char* const sk = smem + buf * 2 * TBYTES;
      const char* const sv = sk + TBYTES;
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        f32x16 s, dp;
        products(sk, sv, k2, s, dp);
        const int k0 = t * MA_KT + k2 * 32;
        const auto at = sc.template at<true>(k0 + lhi * 4 - pos);
        const int ll = ma_opaque(lim - (k0 + lhi * 4));
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
          if (REL && D == 128) __builtin_amdgcn_sched_barrier(0);
          i32x4 dk4 = {dq, dq, dq, dq};
          if (docs && !(fl & 2)) dk4 = *(const i32x4*)(sdoc + buf * MA_KT + k2 * 32 + rg * 8 + lhi * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = rg * 4 + e;
            float sq = 0.f;
            const float pr = sc.template prob<true>(s[r], at, rg * 8 + e, lse2, sq);
            float ds = pr * (dp[r] - delta);
            if (!(fl & 2)) ds = (rg * 8 + e < ll) & (dk4[e] == dq) ? ds : 0.f;
            if (REL) dp[r] = ds;                                   // (kept for the diagonals)
            if (MODE & MA_CAP) ds *= sc.slope(sq);
            s[r] = ds * up;
          }
        }
        if (REL) {
          // distance of the block's first key and first row; its 63 diagonals
          const int dist = k0 - (bs.pos0 + iw);
          if (dist + 31 <= -p.reach || dist - 31 >= p.reach) {
            float f = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) f += dp[r];
            if (dist < 0) far_l += f; else far_r += f;
          } else {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int r = 0; r < 16; ++r) sblk[l31 * 33 + ma_row(r) + 4 * lhi] = dp[r];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int c = lane;                                    // key - row = c - 31
            float f = 0.f;
#pragma unroll 2
            for (int q = 0; q < 32; ++q) {
              const int kk = q + c - 31;
              const float v = sblk[q * 33 + min(max(kk, 0), 31)];
              f += (kk >= 0) & (kk < 32) ? v : 0.f;
            }
            const int dd = dist + c - 31;
            if (c < 63) {
              if (dd <= -p.reach) far_l += f;
              else if (dd >= p.reach) far_r += f;
              else sacc[dd + p.reach] += f;
            }
          }
        }
        v8 pf[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[q * 8 + e];
          pf[q] = ma_pack<T>(x);
        }
        ma_stream<2 * DT, REL && D == 128 ? 2 : 3, v8>([&](auto x) { return TL::template tr_frag<v8>(sk, tbase, x % DT, k2 * 32 + x / DT * 16); },
                                 [&](auto x, const v8 f) { o[x % DT] = ma_mfma(f, pf[x / DT], o[x % DT]); });
      }
    }
    buf ^= 1;
    t = tn; fl = fln;
  }
  float z = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) z += o[dt][r] * 0.f;
  // an infinity or NaN came in, perhaps by a key that the row does not see.  (Where D or lse is not finite, something that it sees was not: all NaN.)
  const unsigned long long bz = __ballot(z != z && delta - delta == 0.f && lse == lse);
  unsigned bad = (unsigned)bz | (unsigned)(bz >> 32);
  if (rok) {
    const float f = p.scale / up;
    T* const out = (T*)p.dQ + b * p.dq_sb + (int64_t)i * p.dq_si + h * p.dq_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int d = dt * 32 + rg * 8 + lhi * 4;
        typedef T t4 __attribute__((ext_vector_type(4)));
        if (d < p.head_dim) *(t4*)(out + d) = t4{(T)(o[dt][rg * 4] * f), (T)(o[dt][rg * 4 + 1] * f), (T)(o[dt][rg * 4 + 2] * f), (T)(o[dt][rg * 4 + 3] * f)};
      }
  }
  if (REL) {
    const int ln = ma_opaque(lane);                    // (the exchange addresses are made here, not kept through the loops)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      far_l += __int_as_float(__builtin_amdgcn_ds_bpermute((ln ^ o) << 2, __float_as_int(far_l)));
      far_r += __int_as_float(__builtin_amdgcn_ds_bpermute((ln ^ o) << 2, __float_as_int(far_r)));
    }
    if (lane == 0) { sacc[0] += far_l; sacc[nrel - 1] += far_r; }
    __syncthreads();
    float* const out = w.rel + ((int64_t)bh * nqb + qb) * nrel;
    const float* const s0 = srel + ma_rel_floats(p.reach) + 32 * 33;
    for (int e = tid; e < nrel; e += 256) {
      float f = 0.f;
#pragma unroll
      for (int ww = 0; ww < 4; ++ww) f += s0[ww * (32 * 33 + nrel) + e];
      out[e] = f;
    }
  }
  while (bad) {
    const int r = __builtin_ctz(bad);
    bad &= bad - 1;
    if (iw + r < p.Nq) ma_slow_dq<T>(ma_late_args(), b, h, iw + r, __shfl(lse2, r, 64), __shfl(delta, r, 64));
  }
}

// dRel[h][e] = sum over batch rows and row blocks of the partial rows, fp64, in order
__global__ __launch_bounds__(256) void ma_rel_sum_kernel(const float* part, float* out, const int batch, const int heads, const int nqb, const int nrel) {
  const int e = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (e >= nrel) return;
  double t = 0.;
  for (int b = 0; b < batch; ++b)
    for (int q = 0; q < nqb; ++q) t += (double)part[(((int64_t)b * heads + h) * nqb + q) * nrel + e];
  out[(int64_t)h * nrel + e] = (float)t;
}

// ---- dK, dV ---------------------------------------------------------------------------------------------------------------------------------
// block: 4 waves x 32 keys.  K fragments stay in registers; V's too at D = 64, at D = 128 they are read again from LDS (both accumulators take
// 128 registers there).  Q / dO tiles of ROWS rows by DMA into two buffers.
template <typename T, int D, int MODE>
__global__ __launch_bounds__(256, 2) void ma_dkv_kernel(const MgldMaskAttn p, const GradWork w, const int nkb, const int nsp) {
  typedef typename MaVec<T>::v8 v8;
  typedef Tile<D> TL;
  constexpr int DK = D / 16, DT = D / 32, ROWS = D == 64 ? 64 : 32, NH = ROWS / 32;
  constexpr bool VLDS = D == 128;
  constexpr int AHEAD = D == 128 ? 3 : 4;          // operands on their way
  constexpr int TBYTES = ROWS * TL::RB, STAT = 3 * MA_KT * 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];      // [2] x {Q, dO}, [2] x {lse, delta, doc numbers} [64], D = 128: V of the block's keys; the distance rows
  char* const sstat = smem + 4 * TBYTES;
  char* const sV = sstat + 2 * STAT;
  float* const srel = (float*)(sV + (VLDS ? 128 * TL::RB : 0));
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, lhi = lane >> 5;
  const int G = p.heads / p.kv_heads, nbk = p.batch * p.kv_heads;
  const int per_kb = nbk * nsp;
  const int kb = blockIdx.x / per_kb;                               // (the first key blocks have the most rows under a causal mask: they come first)
  int rem = blockIdx.x % per_kb;
  const int split = rem / nbk;
  rem %= nbk;
  const int b = rem / p.kv_heads, hk = rem % p.kv_heads;
  const int j0 = kb * 128, jw = j0 + wave * 32;
  const BatchSpan bs(p, b);
  const bool docs = p.doc_q != nullptr;
  // each query with a document sees its own key: only padding rows are blind.  (Asking every row's lse cost 40 of 500 us on 4096 packed tokens.)
  const bool own = p.doc_q == p.doc_k && p.doc_q_sb == p.doc_k_sb && bs.pos0 == 0;
  const int ntk = ma_tiles(p.Nkv), ntq = ma_tiles(p.Nq);
  const i32x4* const qdoc = w.doc + (int64_t)p.batch * ntk + (int64_t)b * ntq;
  const int d8 = p.head_dim / 8;
  v8 zero;
#pragma unroll
  for (int e = 0; e < 8; ++e) zero[e] = (T)0.f;
  const int j = jw + l31;
  const int dj = docs && j < bs.len ? p.doc_k[b * p.doc_k_sb + j] : -1;
  const bool jok = j < bs.len && (!docs || dj >= 0);                // keys that may be seen; the others hold anything
  int bmin = 0, bmax = -1, wmin = 0, wmax = -1;
  bool buni = false, wuni = false;
  if (docs) {
    ma_doc_range(p.doc_k + b * p.doc_k_sb, j0, min(j0 + 128, bs.len), bmin, bmax, buni);
    ma_doc_range(p.doc_k + b * p.doc_k_sb, jw, min(jw + 32, bs.len), wmin, wmax, wuni);
  }
  const T* const Kr = (const T*)p.K + b * p.k_sb + hk * p.k_sh + (int64_t)j * p.k_si;
  const T* const Vr = (const T*)p.V + b * p.v_sb + hk * p.v_sh + (int64_t)j * p.v_si;
  v8 kf[DK], vf[VLDS ? 1 : DK];
#pragma unroll
  for (int ks = 0; ks < DK; ++ks) {
    const bool ok = jok && ks * 2 + lhi < d8;
    kf[ks] = ok ? *(const v8*)(Kr + ks * 16 + lhi * 8) : zero;
    const v8 v = ok ? *(const v8*)(Vr + ks * 16 + lhi * 8) : zero;
    if constexpr (VLDS) *(v8*)(sV + TL::chunk_at(wave * 32 + l31, ks * 2 + lhi)) = v;        // (read back by this wave only)
    else vf[ks] = v;
  }
  if (MODE & MA_REL) ma_load_rel(p, hk * G, G, srel);
  constexpr bool F16 = __is_same(T, f16);
  const float pup = F16 ? 10.f : 0.f;                                // fp16: P is rounded as 2^10 P
  const float gup = F16 ? ma_pow2_to(w.gmax[0], MA_DS_EXP) * 9.765625e-4f : 1.f;       // (P carries 2^10 already)

  // tiles of 64 rows that some key of the block / of the wave is seen from, for every head of the group; dealt to the nsp blocks in turn
  int w0 = -64, g = 0, turn = 0, half = NH == 2 ? 0 : 1, cur = -1, curf = 0;
  unsigned long long act = 0, wact = 0, wfull = 0, pads = 0;
  auto advance = [&](int& flags, int& head) __attribute__((always_inline)) {        // first row of the next stage, or -1
    if (NH == 1 && half == 0 && cur * MA_KT + 32 < p.Nq) { half = 1; flags = curf; head = g; return cur * MA_KT + 32; }
    for (;;) {
      while (!act) {
        w0 += 64;
        if (w0 >= ntq) { if (++g >= G) return -1; w0 = 0; }
        const int t = w0 + lane, ia = t * MA_KT, ib = min(ia + MA_KT, p.Nq) - 1;
        bool a = t < ntq && bs.limit(p, bs.pos0 + ib) > j0, wa = t < ntq && bs.limit(p, bs.pos0 + ib) > jw, pad = bs.limit(p, bs.pos0 + ia) <= 0;
        bool f = wa && ia + MA_KT <= p.Nq && bs.limit(p, bs.pos0 + ia) >= jw + 32;
        if (docs) {
          const i32x4 dt = t < ntq ? qdoc[t] : i32x4{0x7fffffff, -1, 0, 0};
          a = a && dt[0] <= bmax && dt[1] >= bmin;
          wa = wa && dt[0] <= wmax && dt[1] >= wmin;
          f = f && wa && dt[2] && wuni && dt[0] == wmin;
          pad = pad || (own && ib < bs.len ? dt[3] != 0 : !f);
        }
        act = __ballot(a);
        wact = __ballot(a && wa);
        wfull = __ballot(a && f);
        pads = __ballot(pad);
      }
      const int c = __builtin_ctzll(act);
      act &= act - 1;
      const bool mine = turn == split;
      turn = turn + 1 == nsp ? 0 : turn + 1;
      if (!mine) continue;
      cur = __builtin_amdgcn_readfirstlane(w0 + c); half = 0;
      flags = curf = (int)((wact >> c) & 1) | (int)((wfull >> c) & 1) << 1 | (int)((pads >> c) & 1) << 2;
      head = g;
      return cur * MA_KT;
    }
  };
  const TileDma<D, ROWS, 4> dq(wave, lane, p.q_si, p.head_dim), dg(wave, lane, p.do_si, p.head_dim);
  const unsigned lds0 = ma_lds_addr(smem);
  auto load_stage = [&](const int i0, const int gg, const int buf, const int flags) __attribute__((always_inline)) {
    const int h = hk * G + gg;
    const unsigned a = lds0 + buf * 2 * TBYTES, st = lds0 + 4 * TBYTES + buf * STAT;
    const int32_t* const ids = docs ? p.doc_q + b * p.doc_q_sb + i0 : nullptr;
    const int64_t row = ((int64_t)b * p.heads + h) * p.Nq + i0;
    const float* const lse = p.lse + row;
    auto blind = [&](const int r) __attribute__((always_inline)) { return lse[r] == -MA_INF; };       // rows that see nothing hold anything
    dq.load((const T*)p.Q + b * p.q_sb + h * p.q_sh, (int64_t)i0 * p.q_si * 2, p.q_si, p.Nq - i0, a, flags & 4, blind);
    dg.load((const T*)p.dO + b * p.do_sb + h * p.do_sh, (int64_t)i0 * p.do_si * 2, p.do_si, p.Nq - i0, a + TBYTES, flags & 4, blind);
    if (wave == 0) ma_dma4(st, lane, p.Nq - i0, p.lse + row);
    if (wave == 1) ma_dma4(st + 256, lane, p.Nq - i0, w.delta + row);
    if (wave == 2 && docs) ma_dma4(st + 512, lane, p.Nq - i0, ids);
  };

  f32x16 ok_[DT], ov[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) { ok_[dt] = ma_zero(); ov[dt] = ma_zero(); }
  const int rbase = TL::row_base(lane), tbase = TL::tr_base(lane);
  int fl = 0, fln = 0, hd = 0, hdn = 0, buf = 0;
  int i0 = advance(fl, hd);
  if (i0 >= 0) load_stage(i0, hd, 0, fl);
  while (i0 >= 0) {
    ma_dma_wait();
    __syncthreads();
    const int in = advance(fln, hdn);
    if (in >= 0) load_stage(in, hdn, buf ^ 1, fln);
    if (fl & 1) {
      const char* const sq_ = smem + buf * 2 * TBYTES;
      const char* const sg = sq_ + TBYTES;
      const float* const sl = (const float*)(sstat + buf * STAT);
      const int rb = D == 128 ? ma_opaque(rbase) : rbase, tb = D == 128 ? ma_opaque(tbase) : tbase;      // (registers: the swizzled addresses are made per stage)
      const Score<MODE> sc(p, hk * G + hd, srel + hd * ma_rel_floats(p.reach));
#pragma unroll
      for (int q2 = 0; q2 < NH; ++q2) {
        f32x16 s = ma_zero(), dp = ma_zero();
        if constexpr (VLDS) {                                       // Q, dO and V fragments in turn
          v8 vr;
          ma_stream<3 * DK, AHEAD, v8>([&](auto x) { return x % 3 == 0 ? TL::template row_frag<v8>(sq_, rb, q2 * 32, x / 3) : x % 3 == 1 ? TL::template row_frag<v8>(sV, rb, wave * 32, x / 3)
                                                                                                                                     : TL::template row_frag<v8>(sg, rb, q2 * 32, x / 3); },
                                       [&](auto x, const v8 f) { if (x % 3 == 0) s = ma_mfma(f, kf[x / 3], s); else if (x % 3 == 1) vr = f; else dp = ma_mfma(f, vr, dp); });
        } else {
          ma_stream<2 * DK, AHEAD, v8>([&](auto x) { return TL::template row_frag<v8>(x & 1 ? sg : sq_, rb, q2 * 32, x >> 1); },
                                       [&](auto x, const v8 f) { if (x & 1) dp = ma_mfma(f, vf[x >> 1], dp); else s = ma_mfma(f, kf[x >> 1], s); });
        }
        const int ib = i0 + q2 * 32;
        const auto at = sc.template at<false>(j - (bs.pos0 + ib + lhi * 4));
        const int il = ma_opaque(ib + lhi * 4);
        v8 pf[4];                                                   // P, then dT
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
          if (D == 128 && MODE) __builtin_amdgcn_sched_barrier(0);        // (four scores at a time: more in flight spill)
          const int rr = q2 * 32 + rg * 8 + lhi * 4;
          const f32x4 lse2 = *(const f32x4*)(sl + rr) * MA_LOG2E, delta = *(const f32x4*)(sl + 64 + rr);
          i32x4 di = {dj, dj, dj, dj};
          if (docs && !(fl & 2)) di = *(const i32x4*)((const int*)sl + 128 + rr);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = rg * 4 + e;
            float sq = 0.f;
            float pr = sc.template prob<false>(s[r], at, rg * 8 + e, lse2[e] - pup, sq);
            float ds = pr * (dp[r] - delta[e]) * gup;
            if (MODE & MA_CAP) ds *= sc.slope(sq);
            if (!(fl & 2)) {
              const int i = il + rg * 8 + e;
              const bool vis = jok & (i < p.Nq) & (j < bs.limit(p, bs.pos0 + i)) & (di[e] == dj);
              pr = vis ? pr : 0.f;
              ds = vis ? ds : 0.f;
            }
            pf[rg >> 1][(rg & 1) * 4 + e] = (T)pr;                  // rounded to nearest: maskattn.h, ma_pack
            pf[2 + (rg >> 1)][(rg & 1) * 4 + e] = (T)ds;
          }
        }
        ma_stream<4 * DT, 3, v8>([&](auto x) { return TL::template tr_frag<v8>(x & 1 ? sq_ : sg, tb, (x >> 1) % DT, q2 * 32 + x / (2 * DT) * 16); },
                                 [&](auto x, const v8 f) {
                                   if (x & 1) ok_[(x >> 1) % DT] = ma_mfma(f, pf[2 + x / (2 * DT)], ok_[(x >> 1) % DT]);
                                   else ov[(x >> 1) % DT] = ma_mfma(f, pf[x / (2 * DT)], ov[(x >> 1) % DT]);
                                 });
      }
    }
    buf ^= 1;
    i0 = in; fl = fln; hd = hdn;
  }
  if (j >= p.Nkv) return;
  const float fv = F16 ? 9.765625e-4f : 1.f, fk = p.scale * fv / gup;
  if (nsp > 1) {
    float* const out = w.kv + ((((int64_t)split * p.batch + b) * p.Nkv + j) * p.kv_heads + hk) * 2 * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int d = dt * 32 + rg * 8 + lhi * 4;
        *(f32x4*)(out + d) = f32x4{ok_[dt][rg * 4], ok_[dt][rg * 4 + 1], ok_[dt][rg * 4 + 2], ok_[dt][rg * 4 + 3]} * fk;
        *(f32x4*)(out + D + d) = f32x4{ov[dt][rg * 4], ov[dt][rg * 4 + 1], ov[dt][rg * 4 + 2], ov[dt][rg * 4 + 3]} * fv;
      }
    return;
  }
  T* const okp = (T*)p.dK + b * p.dk_sb + (int64_t)j * p.dk_si + hk * p.dk_sh;
  T* const ovp = (T*)p.dV + b * p.dv_sb + (int64_t)j * p.dv_si + hk * p.dv_sh;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      const int d = dt * 32 + rg * 8 + lhi * 4;
      typedef T t4 __attribute__((ext_vector_type(4)));
      if (d < p.head_dim) {
        *(t4*)(okp + d) = t4{(T)(ok_[dt][rg * 4] * fk), (T)(ok_[dt][rg * 4 + 1] * fk), (T)(ok_[dt][rg * 4 + 2] * fk), (T)(ok_[dt][rg * 4 + 3] * fk)};
        *(t4*)(ovp + d) = t4{(T)(ov[dt][rg * 4] * fv), (T)(ov[dt][rg * 4 + 1] * fv), (T)(ov[dt][rg * 4 + 2] * fv), (T)(ov[dt][rg * 4 + 3] * fv)};
      }
    }
}

// dK, dV = the sum of the nsp partial results, in order; four elements per thread
template <typename T, int D>
__global__ __launch_bounds__(256) void ma_kv_sum_kernel(const MgldMaskAttn p, const float* part, const int nsp, const int64_t n4) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= n4) return;
  const int e = (int)(x % (2 * D / 4)) * 4;
  const int64_t row = x / (2 * D / 4);                              // (b, j, hk)
  const int hk = (int)(row % p.kv_heads), d = e % D;
  const int64_t bj = row / p.kv_heads;
  const int j = (int)(bj % p.Nkv), b = (int)(bj / p.Nkv);
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < nsp; ++s) t += *(const f32x4*)(part + (int64_t)s * n4 * 4 + x * 4);
  if (d >= p.head_dim) return;
  T* const out = e < D ? (T*)p.dK + b * p.dk_sb + (int64_t)j * p.dk_si + hk * p.dk_sh : (T*)p.dV + b * p.dv_sb + (int64_t)j * p.dv_si + hk * p.dv_sh;
  typedef T t4 __attribute__((ext_vector_type(4)));
  *(t4*)(out + d) = t4{(T)t[0], (T)t[1], (T)t[2], (T)t[3]};
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------------
int64_t up256(const int64_t n) { return (n + 255) / 256 * 256; }
struct GradPlan {
  int nsp, nqb, nkb;
  int64_t rows, doc, delta, amax, gmax, rel, kv, total;      // byte offsets
};
GradPlan grad_plan(const MgldMaskAttn* p) {
  GradPlan g;
  const int D = p->head_dim <= 64 ? 64 : 128;
  g.rows = (int64_t)p->batch * p->heads * p->Nq;
  g.nqb = (p->Nq + 127) / 128;
  g.nkb = (p->Nkv + 127) / 128;
  const int64_t blocks = (int64_t)g.nkb * p->batch * p->kv_heads, items = (int64_t)(p->heads / p->kv_heads) * ma_tiles(p->Nq);
  int64_t n = blocks > 0 ? 512 / blocks : 1;                        // two blocks per CU
  if (n > (items + 3) / 4) n = (items + 3) / 4;
  g.nsp = n < 1 ? 1 : n > 8 ? 8 : (int)n;
  g.doc = 0;
  g.delta = up256(ma_doc_bytes(p));
  g.amax = g.delta + up256(g.rows * 4);
  g.gmax = g.amax + (p->bf16 ? 0 : up256((int64_t)p->batch * p->heads * g.nqb * 16));
  g.rel = g.gmax + 256;
  g.kv = g.rel + (p->dRel ? up256(g.rows ? (int64_t)p->batch * p->heads * g.nqb * (2 * p->reach + 1) * 4 : 0) : 0);
  g.total = g.kv + (g.nsp > 1 ? (int64_t)g.nsp * p->batch * p->Nkv * p->kv_heads * 2 * D * 4 : 0);
  return g;
}

template <typename K>
void grad_lds(K kernel, const int lds) {
  if (lds > 64 * 1024) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <typename T, int D, int MODE>
int grad_launch(const MgldMaskAttn& p, hipStream_t st) {
  const GradPlan g = grad_plan(&p);
  char* const wk = (char*)p.work;
  GradWork w;
  w.doc = (const i32x4*)(wk + g.doc);
  w.delta = (float*)(wk + g.delta);
  w.amax = p.bf16 ? nullptr : (float*)(wk + g.amax);
  w.gmax = (float*)(wk + g.gmax);
  w.rel = (float*)(wk + g.rel);
  w.kv = (float*)(wk + g.kv);
  const int nrel = p.rel ? 2 * p.reach + 1 : 0, next = p.rel ? ma_rel_floats(p.reach) : 0, G = p.heads / p.kv_heads;
  MGLD_REQUIRE((int64_t)g.nqb * p.batch * p.heads <= 0x7fffffff && (int64_t)g.nkb * p.batch * p.kv_heads * g.nsp <= 0x7fffffff,
               "masked_attention_grad: grid");
  if (p.doc_q) {
    const int rc = ma_doc_tiles(p, wk + g.doc, st);
    if (rc) return rc;
  }
  if (p.Nq > 0) {
    const dim3 grid((unsigned)((int64_t)g.nqb * p.batch * p.heads));
    const int lds = 4 * MA_KT * Tile<D>::RB + 2 * MA_KT * 4 + next * 4;
    if constexpr (MODE & MA_REL) {
      if (p.dRel) {
        const int lr = lds + 4 * (32 * 33 + nrel) * 4;
        grad_lds(ma_dq_kernel<T, D, MODE, true>, lr);
        ma_dq_kernel<T, D, MODE, true><<<grid, 256, lr, st>>>(p, w, g.nqb);
      }
    }
    if (!(MODE & MA_REL) || !p.dRel) {
      grad_lds(ma_dq_kernel<T, D, MODE, false>, lds);
      ma_dq_kernel<T, D, MODE, false><<<grid, 256, lds, st>>>(p, w, g.nqb);
    }
  }
  if (w.amax) ma_amax_kernel<<<1, 1024, 0, st>>>(w.amax, (int64_t)p.batch * p.heads * g.nqb * 4, w.gmax);
  if (p.dRel) ma_rel_sum_kernel<<<dim3(cdiv(nrel, 256), p.heads), 256, 0, st>>>(w.rel, p.dRel, p.batch, p.heads, g.nqb, nrel);
  if (p.Nkv > 0) {
    constexpr int ROWS = D == 64 ? 64 : 32;
    const int lds = 4 * ROWS * Tile<D>::RB + 2 * 3 * MA_KT * 4 + (D == 128 ? 128 * Tile<D>::RB : 0) + G * next * 4;
    grad_lds(ma_dkv_kernel<T, D, MODE>, lds);
    const int64_t nb = (int64_t)g.nkb * p.batch * p.kv_heads * g.nsp;
    ma_dkv_kernel<T, D, MODE><<<dim3((unsigned)nb), 256, lds, st>>>(p, w, g.nkb, g.nsp);
    if (g.nsp > 1) {
      const int64_t n4 = (int64_t)p.batch * p.Nkv * p.kv_heads * 2 * D / 4;
      MGLD_REQUIRE((n4 + 255) / 256 <= 0x7fffffff, "masked_attention_grad: grid");
      ma_kv_sum_kernel<T, D><<<dim3((unsigned)((n4 + 255) / 256)), 256, 0, st>>>(p, w.kv, g.nsp, n4);
    }
  }
  return mgld_check_launch("masked_attention_grad");
}
}  // namespace

extern "C" int64_t mgld_masked_attention_grad_work(const MgldMaskAttn* p) {
  if (!p || ma_check(p, true) || p->batch == 0) return 0;
  return grad_plan(p).total;
}

extern "C" int mgld_masked_attention_grad(const MgldMaskAttn* p, void* stream) {
  const int rc = ma_check(p, true);
  if (rc) return rc;
  MGLD_REQUIRE(!p->dRel || p->rel, "masked_attention_grad: dRel without rel");
  hipStream_t st = (hipStream_t)stream;
  if (p->batch == 0) {
    if (!p->dRel) return MGLD_OK;
    ma_rel_sum_kernel<<<dim3(cdiv(2 * p->reach + 1, 256), p->heads), 256, 0, st>>>(nullptr, p->dRel, 0, p->heads, 0, 2 * p->reach + 1);
    return mgld_check_launch("masked_attention_grad");
  }
  const int64_t need = mgld_masked_attention_grad_work(p);
  MGLD_REQUIRE(p->work && (uintptr_t)p->work % 16 == 0 && p->work_bytes >= need, "masked_attention_grad: work buffer too small");
  MA_DISPATCH(grad_launch, p, st)
}
