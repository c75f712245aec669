// pp_common.h — device helpers of the ping-pong GEMM family (ppgemm.hip: LINEAR, conv3r.hip: patch-staged 3x3 convolutions).
//
// Structure shared by both kernels (gfx950, one 512-thread workgroup per CU):
//   * eight waves in two GROUPS of four (group = wave >> 2: one wave of each group per SIMD).  A K slice of 32 is one PHASE; every phase is
//     [L: ds_read_b128 the phase's fragments + issue LDS-DMA pieces of a later stage] s_barrier [M: the phase's MFMAs] s_barrier.  Group 1
//     runs ONE barrier behind group 0, so on every SIMD one wave is in its matrix section while the other reads LDS and issues DMA: the
//     matrix pipe alternates between the two waves instead of both waiting at the same stage barrier (the 128-class structure of
//     igemm.hip / conv3q.hip: matrix pipe 40 % busy, waves parked 44 % on the per-stage barrier, profiles/r03_pmc_conv3q.txt).
//   * operands reach LDS by `buffer_load_dwordx4 ... offen lds` (LDS-DMA through a buffer descriptor: one 32-bit VGPR offset per lane,
//     everything else scalar) into a ring of stages; waits are COUNTED (`s_waitcnt vmcnt(n)`, n = the pieces of the newer stages this
//     wave has issued) and sit one phase before the first read of the stage; barriers are raw `s_barrier` (no vmcnt drain).
//   * v_mfma_f32_16x16x32_f16: wave tiles are any multiple of 16 (the N = 320 layers take 80-column wave tiles), one ds_read_b128 per
//     16-row fragment and phase.  The WEIGHT fragment is the first operand: a lane ends up with 4 consecutive output channels of one
//     output row per fragment, adjacent fragments are paired by v_permlane16_swap into 8 consecutive channels = one 16-byte store.
//   * the epilogue runs from registers (no LDS patch, no barrier): bias / per-frame row vector / SiLU or GEGLU / alpha, beta * residual.
#pragma once
#include "igemm_common.h"

namespace {

// (hipcc parses kernel bodies in its HOST pass too; the buffer-resource builtins do not exist there, and a kernel template whose body
// fails that way silently loses its launch stub.  The host pass therefore sees empty stand-ins — device code is unaffected.)
#if defined(__HIP_DEVICE_COMPILE__)
typedef __amdgpu_buffer_rsrc_t pp_rsrc_t;
__device__ __forceinline__ pp_rsrc_t pp_make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00020000);
}
// one 1-KiB LDS-DMA piece: lane l's 16 bytes at base + voff + soff land at lds + 16 l
__device__ __forceinline__ void pp_dma16(const pp_rsrc_t rsrc, char* lds_wave_base, const uint32_t voff, const uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds_wave_base, 16, voff, __builtin_amdgcn_readfirstlane(soff), 0, 0);
}
#else
typedef const void* pp_rsrc_t;
__device__ __forceinline__ pp_rsrc_t pp_make_rsrc(const void* base, uint32_t) { return base; }
__device__ __forceinline__ void pp_dma16(const pp_rsrc_t, char*, const uint32_t, const uint32_t) {}
#endif

template <int N>
__device__ __forceinline__ void pp_wait_vm() {
  static_assert(N >= 0 && N <= 63, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pp_wait_lgkm0() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void pp_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// ---- epilogue from registers --------------------------------------------------------------------------------------------
// acc[ni][mi]: fragment (weight rows n0 + 16 ni .., output rows m0 + 16 mi ..): lane l holds output row (l & 15), channels 4 (l >> 4) + r.
// EPI: 0 = bias / rowvec / none or SiLU / alpha / residual; 1 = GEGLU (the wave's 64 weight rows are [32 value | 32 gate] of 32 outputs).
struct PPEpi {
  const float* bias; const float* rowvec; const f16* R; f16* C;
  const f16* Rlo; f16* Clo;    // low planes of the residual / the output (MgldIGemm.Rlo / Clo), or null
  // LayerNorm folded into this projection (MgldIGemm.ln_part): out = act(rstd_m (acc - mean_m s_n) + bias_n); ln_M = rows of one chunk of ln_part
  const float* ln_part = nullptr; const float* ln_s = nullptr; int ln_chunks = 0, ln_M = 0; float ln_invK = 0.f, ln_eps = 0.f;
  // row statistics of what this tile stores (MgldIGemm.row_part): this WAVE's slot of the block table in LDS, [BM rows][2] floats, or null
  float* row_tab = nullptr;
  int rows_per_frame, ld_rowvec, ldr, ldc, act; float alpha, beta;
  bool noswap;     // A/B and bring-up: every fragment by 8-byte stores (no v_permlane16_swap pairing)
};

// FEAT: the round-6 extras (stream low planes, folded LayerNorm, row statistics) are compiled in; callers branch ONCE per block on whether any of
// them is set, so a plain launch runs the round-5 instruction stream (the GEGLU epilogue is VALU-bound: the dormant checks cost it 5 %)
template <int MI, int NI, bool GEGLU, bool FEAT, bool RELU, typename RowFn>
__device__ __forceinline__ void pp_epilogue_(const PPEpi& e, f32x4 (&acc)[NI][MI], const int lane, const int n0, const RowFn row_of) {
  // n0: first output channel (packed weight row for GEGLU) of this wave; row_of(mi) = global output row of this lane in fragment mi, or -1
  const int q = lane >> 4;
  constexpr int NO = GEGLU ? NI / 2 : NI;            // output fragments
  static_assert(!GEGLU || NI == 4, "GEGLU: 64 weight rows per wave");
  const float alpha = e.alpha;
  // per-lane column constants (bias, plus the per-frame row vector of the frame the rows lie in), loaded ONCE per frame: inside the row
  // loop every fragment row paid an L2 round trip for them.  Rows of a tile are almost always one frame.
  f32x4 cv[NI];
  // folded LayerNorm: the column sums s_n.  Narrow wave tiles (the GEGLU tiles: 64 weight rows = 4 fragments) hold them like the bias; wide ones
  // (the 256 x 320 tile: 10 fragments, 250 registers already) re-read them per fragment from L1
  constexpr bool HOIST_S = FEAT && NI <= 4;
  f32x4 sv[HOIST_S ? NI : 1];
  if constexpr (HOIST_S) {
#pragma unroll
    for (int f = 0; f < NI; ++f) sv[f] = e.ln_part ? *(const f32x4*)(e.ln_s + n0 + f * 16 + 4 * q) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int fr_loaded = -2;
  auto load_cv = [&](const int fr) {
#pragma unroll
    for (int f = 0; f < NI; ++f) {
      cv[f] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (e.bias) cv[f] = *(const f32x4*)(e.bias + n0 + f * 16 + 4 * q);
    }
    if (fr >= 0) {
      const float* rv = e.rowvec + (int64_t)fr * e.ld_rowvec + n0 + 4 * q;
#pragma unroll
      for (int f = 0; f < NI; ++f) cv[f] += *(const f32x4*)(rv + f * 16);
    }
    fr_loaded = fr;
  };
  const int nb = GEGLU ? n0 / 2 : n0;                // first output column of the wave
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int m = row_of(mi);
    {
      const int fr = (!GEGLU && e.rowvec && m >= 0) ? m / e.rows_per_frame : -1;
      if (fr != fr_loaded && (m >= 0 || fr_loaded == -2)) load_cv(fr);
    }
    // folded LayerNorm: this row's (mean, rstd) from the producer's chunk sums
    float ln_mu = 0.f, ln_rs = 1.f;
    if (FEAT && e.ln_part && m >= 0) {
      float s1 = 0.f, s2 = 0.f;
      for (int c = 0; c < e.ln_chunks; ++c) {
        const f32x2 t = *(const f32x2*)(e.ln_part + ((int64_t)c * e.ln_M + m) * 2);
        s1 += t[0]; s2 += t[1];
      }
      const float mu = s1 * e.ln_invK;
      ln_rs = __builtin_amdgcn_rsqf(fmaxf(s2 * e.ln_invK - mu * mu, 0.f) + e.ln_eps);
      ln_mu = -mu * ln_rs;                         // rstd (acc - mean s) = acc rstd + (-mean rstd) s: two FMAs per element
    }
    auto ln_of = [&](const f32x4 a, const int f) -> f32x4 {
      if (!FEAT || !e.ln_part) return a;
      f32x4 sn;
      if constexpr (HOIST_S) sn = sv[f];
      else sn = *(const f32x4*)(e.ln_s + n0 + f * 16 + 4 * q);
      return a * ln_rs + ln_mu * sn;
    };
    auto out_frag = [&](const int f) -> f32x4 {      // output fragment f of this row block, epilogue arithmetic applied (not the residual)
      if constexpr (GEGLU) {
        const f32x4 bv = cv[f], bg = cv[2 + f];
        const f32x4 av = ln_of(acc[f][mi], f), ag = ln_of(acc[2 + f][mi], 2 + f);
        const e2 v0 = pk(av[0] + bv[0], av[1] + bv[1]), v1 = pk(av[2] + bv[2], av[3] + bv[3]);
        const e2 g0 = gelu2(pk(ag[0] + bg[0], ag[1] + bg[1])), g1 = gelu2(pk(ag[2] + bg[2], ag[3] + bg[3]));
        const e2 r0 = v0 * g0, r1 = v1 * g1;
        return f32x4{r0[0] * alpha, r0[1] * alpha, r1[0] * alpha, r1[1] * alpha};
      } else {
        f32x4 v = ln_of(acc[f][mi], f) + cv[f];
        if (e.act == MGLD_ACT_SILU) {
          const e2 s0 = silu2(pk(v[0], v[1])), s1 = silu2(pk(v[2], v[3]));
          v = f32x4{s0[0], s0[1], s1[0], s1[1]};
        } else if (RELU && e.act == MGLD_ACT_RELU) {   // SPADE's shared convolution (conv + ReLU); compiled into the convolution's copy only —
                                                       // the runtime check alone put the 256 x 320 LINEAR tile (256 VGPRs) into scratch: 54 -> 70 us
          v = f32x4{fmaxf(v[0], 0.f), fmaxf(v[1], 0.f), fmaxf(v[2], 0.f), fmaxf(v[3], 0.f)};
        }
        return v * alpha;
      }
    };
    float rsum = 0.f, rsq = 0.f;                     // row_tab: this lane's share of row m's (sum, sumsq) over the wave's columns
    auto store4 = [&](const int f) {                 // fragment f by 8-byte stores of 4 channels
      f32x4 a = out_frag(f);
      if (m < 0) return;
      const int n = nb + f * 16 + 4 * q;
      if (e.R) {
        const f16x4 rr = *(const f16x4*)(e.R + (int64_t)m * e.ldr + n);
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] += e.beta * (float)rr[r];
        if (FEAT && e.Rlo) {
          const f16x4 rl = *(const f16x4*)(e.Rlo + (int64_t)m * e.ldr + n);
          const float bl = e.beta * MGLD_LO_SCALE;
#pragma unroll
          for (int r = 0; r < 4; ++r) a[r] += bl * (float)rl[r];
        }
      }
      const f16x4 o = f16x4{(f16)a[0], (f16)a[1], (f16)a[2], (f16)a[3]};
      *(f16x4*)(e.C + (int64_t)m * e.ldc + n) = o;
      if (FEAT && e.Clo) *(f16x4*)(e.Clo + (int64_t)m * e.ldc + n) = f16x4{lo_plane(a[0], o[0]), lo_plane(a[1], o[1]), lo_plane(a[2], o[2]), lo_plane(a[3], o[3])};
      if (FEAT && e.row_tab) {
#pragma unroll
        for (int r = 0; r < 4; ++r) { rsum += a[r]; rsq += a[r] * a[r]; }
      }
    };
    auto row_flush = [&]() {                         // the four lane rows q hold the same output row: add them up, lane row 0 writes the wave's slot
      if (!FEAT || !e.row_tab) return;
      rsum += __shfl_xor(rsum, 16, 64); rsq += __shfl_xor(rsq, 16, 64);
      rsum += __shfl_xor(rsum, 32, 64); rsq += __shfl_xor(rsq, 32, 64);
      if (q == 0) *(f32x2*)(e.row_tab + (mi * 16 + (lane & 15)) * 2) = f32x2{rsum, rsq};
    };
    if (e.noswap) {
#pragma unroll
      for (int f = 0; f < NO; ++f) store4(f);
      row_flush();
      continue;
    }
    // pairs of fragments -> 16-byte stores: after the swap, lane (row q) holds fragment 2 pr + (q & 1), channels 8 (q >> 1) .. + 8
#pragma unroll
    for (int pr = 0; pr < NO / 2; ++pr) {
      f32x4 a = out_frag(2 * pr), b = out_frag(2 * pr + 1);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[r]), __float_as_uint(b[r]), false, false);
        a[r] = __uint_as_float(s[0]); b[r] = __uint_as_float(s[1]);
      }
      if (m < 0) continue;
      const int n = nb + (2 * pr + (q & 1)) * 16 + (q >> 1) * 8;
      if (e.R) {
        const f16x8 rr = *(const f16x8*)(e.R + (int64_t)m * e.ldr + n);
#pragma unroll
        for (int r = 0; r < 4; ++r) { a[r] += e.beta * (float)rr[r]; b[r] += e.beta * (float)rr[4 + r]; }
        if (FEAT && e.Rlo) {
          const f16x8 rl = *(const f16x8*)(e.Rlo + (int64_t)m * e.ldr + n);
          const float bl = e.beta * MGLD_LO_SCALE;
#pragma unroll
          for (int r = 0; r < 4; ++r) { a[r] += bl * (float)rl[r]; b[r] += bl * (float)rl[4 + r]; }
        }
      }
      const f16x8 o = f16x8{(f16)a[0], (f16)a[1], (f16)a[2], (f16)a[3], (f16)b[0], (f16)b[1], (f16)b[2], (f16)b[3]};
      *(f16x8*)(e.C + (int64_t)m * e.ldc + n) = o;
      if (FEAT && e.Clo)
        *(f16x8*)(e.Clo + (int64_t)m * e.ldc + n) = f16x8{lo_plane(a[0], o[0]), lo_plane(a[1], o[1]), lo_plane(a[2], o[2]), lo_plane(a[3], o[3]),
                                                          lo_plane(b[0], o[4]), lo_plane(b[1], o[5]), lo_plane(b[2], o[6]), lo_plane(b[3], o[7])};
      if (FEAT && e.row_tab) {
#pragma unroll
        for (int r = 0; r < 4; ++r) { rsum += a[r] + b[r]; rsq += a[r] * a[r] + b[r] * b[r]; }
      }
    }
    if constexpr (NO & 1) store4(NO - 1);            // unpaired last fragment
    row_flush();
  }
}

template <int MI, int NI, bool GEGLU, bool RELU = false, typename RowFn>
__device__ __forceinline__ void pp_epilogue(const PPEpi& e, f32x4 (&acc)[NI][MI], const int lane, const int n0, const RowFn row_of) {
  if (e.Rlo || e.Clo || e.ln_part || e.row_tab) pp_epilogue_<MI, NI, GEGLU, true, RELU>(e, acc, lane, n0, row_of);
  else pp_epilogue_<MI, NI, GEGLU, false, RELU>(e, acc, lane, n0, row_of);
}

// ---- the same epilogue + per-channel (sum, sumsq) of the output values (GroupNorm statistics of the output, MgldIGemm.gn_part) ----
// For tiles whose rows lie in ONE frame (`fr`, -1 without a row vector).  Fragment pairs outermost: 16 running sums per lane and pair, reduced
// over the 16 rows of a lane row by DPP adds (quad xor 1, xor 2, half-row mirror, row mirror), then written by lane row heads to this wave's
// slot of the block's LDS table: wave_sums[channel of the wave tile][2].  The caller adds the wave rows up (pp_stats_flush).
__device__ __forceinline__ float pp_row16_sum(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));    // quad_perm [1, 0, 3, 2]
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));    // quad_perm [2, 3, 0, 1]
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));   // row_half_mirror
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));   // row_mirror
#endif
  return v;
}

template <int MI, int NI, bool RELU = false, typename RowFn>
__device__ __forceinline__ void pp_epilogue_stats(const PPEpi& e, f32x4 (&acc)[NI][MI], const int lane, const int n0, const int fr,
                                                  const RowFn row_of, float* __restrict__ wave_sums) {
  const int q = lane >> 4, l15 = lane & 15;
  const float alpha = e.alpha;
  f32x4 cv[NI];
#pragma unroll
  for (int f = 0; f < NI; ++f) {
    cv[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (e.bias) cv[f] = *(const f32x4*)(e.bias + n0 + f * 16 + 4 * q);
  }
  if (fr >= 0) {
    const float* rv = e.rowvec + (int64_t)fr * e.ld_rowvec + n0 + 4 * q;
#pragma unroll
    for (int f = 0; f < NI; ++f) cv[f] += *(const f32x4*)(rv + f * 16);
  }
  auto out_frag = [&](const int f, const int mi) -> f32x4 {
    f32x4 v = acc[f][mi] + cv[f];
    if (e.act == MGLD_ACT_SILU) {
      const e2 s0 = silu2(pk(v[0], v[1])), s1 = silu2(pk(v[2], v[3]));
      v = f32x4{s0[0], s0[1], s1[0], s1[1]};
    } else if (RELU && e.act == MGLD_ACT_RELU) {
      v = f32x4{fmaxf(v[0], 0.f), fmaxf(v[1], 0.f), fmaxf(v[2], 0.f), fmaxf(v[3], 0.f)};
    }
    return v * alpha;
  };
#pragma unroll
  for (int pr = 0; pr < NI / 2; ++pr) {
    e2 ss[4], qq[4];                                             // fp32 pairs
#pragma unroll
    for (int r = 0; r < 4; ++r) { ss[r] = pk(0.f, 0.f); qq[r] = pk(0.f, 0.f); }
    const int nl = (2 * pr + (q & 1)) * 16 + (q >> 1) * 8;       // this lane's 8 channels of the wave tile after the swap
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const int m = row_of(mi);
      f32x4 a = out_frag(2 * pr, mi), b = out_frag(2 * pr + 1, mi);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[r]), __float_as_uint(b[r]), false, false);
        a[r] = __uint_as_float(s[0]); b[r] = __uint_as_float(s[1]);
      }
      if (m < 0) continue;
      if (e.R) {
        const f16x8 rr = *(const f16x8*)(e.R + (int64_t)m * e.ldr + n0 + nl);
#pragma unroll
        for (int r = 0; r < 4; ++r) { a[r] += e.beta * (float)rr[r]; b[r] += e.beta * (float)rr[4 + r]; }
        if (e.Rlo) {
          const f16x8 rl = *(const f16x8*)(e.Rlo + (int64_t)m * e.ldr + n0 + nl);
          const float bl = e.beta * MGLD_LO_SCALE;
#pragma unroll
          for (int r = 0; r < 4; ++r) { a[r] += bl * (float)rl[r]; b[r] += bl * (float)rl[4 + r]; }
        }
      }
      const f16x8 o = f16x8{(f16)a[0], (f16)a[1], (f16)a[2], (f16)a[3], (f16)b[0], (f16)b[1], (f16)b[2], (f16)b[3]};
      *(f16x8*)(e.C + (int64_t)m * e.ldc + n0 + nl) = o;
      if (e.Clo)
        *(f16x8*)(e.Clo + (int64_t)m * e.ldc + n0 + nl) = f16x8{lo_plane(a[0], o[0]), lo_plane(a[1], o[1]), lo_plane(a[2], o[2]), lo_plane(a[3], o[3]),
                                                                lo_plane(b[0], o[4]), lo_plane(b[1], o[5]), lo_plane(b[2], o[6]), lo_plane(b[3], o[7])};
      // (sums of the fp32 values before their rounding to fp16: the zero-mean rounding noise moves mean and variance of >= 10^4 elements
      //  by ~1e-7 relative — the conversions back would cost a third of this block's arithmetic)
      const e2 v[4] = {pk(a[0], a[1]), pk(a[2], a[3]), pk(b[0], b[1]), pk(b[2], b[3])};
#pragma unroll
      for (int r = 0; r < 4; ++r) { ss[r] += v[r]; qq[r] += v[r] * v[r]; }
    }
    float s1[8], q1[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) { s1[r] = pp_row16_sum(ss[r >> 1][r & 1]); q1[r] = pp_row16_sum(qq[r >> 1][r & 1]); }
    if (l15 == 0) {
#pragma unroll
      for (int r = 0; r < 8; r += 2) *(f32x4*)(wave_sums + (nl + r) * 2) = f32x4{s1[r], q1[r], s1[r + 1], q1[r + 1]};
    }
  }
  if constexpr (NI & 1) {                                      // unpaired last fragment: 4 channels per lane
    constexpr int f = NI - 1;
    float ss[4], qq[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) { ss[r] = 0.f; qq[r] = 0.f; }
    const int nl = f * 16 + 4 * q;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const int m = row_of(mi);
      f32x4 a = out_frag(f, mi);
      if (m < 0) continue;
      if (e.R) {
        const f16x4 rr = *(const f16x4*)(e.R + (int64_t)m * e.ldr + n0 + nl);
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] += e.beta * (float)rr[r];
        if (e.Rlo) {
          const f16x4 rl = *(const f16x4*)(e.Rlo + (int64_t)m * e.ldr + n0 + nl);
          const float bl = e.beta * MGLD_LO_SCALE;
#pragma unroll
          for (int r = 0; r < 4; ++r) a[r] += bl * (float)rl[r];
        }
      }
      const f16x4 o = f16x4{(f16)a[0], (f16)a[1], (f16)a[2], (f16)a[3]};
      *(f16x4*)(e.C + (int64_t)m * e.ldc + n0 + nl) = o;
      if (e.Clo) *(f16x4*)(e.Clo + (int64_t)m * e.ldc + n0 + nl) = f16x4{lo_plane(a[0], o[0]), lo_plane(a[1], o[1]), lo_plane(a[2], o[2]), lo_plane(a[3], o[3])};
#pragma unroll
      for (int r = 0; r < 4; ++r) { ss[r] += a[r]; qq[r] += a[r] * a[r]; }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) { ss[r] = pp_row16_sum(ss[r]); qq[r] = pp_row16_sum(qq[r]); }
    if (l15 == 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) { wave_sums[(nl + r) * 2] = ss[r]; wave_sums[(nl + r) * 2 + 1] = qq[r]; }
    }
  }
}

// block table [WGM wave rows][BN][2] in LDS -> part[tile][2][N] (after a block barrier; all 512 threads call)
template <int WGM, int BN>
__device__ __forceinline__ void pp_stats_flush(const float* __restrict__ table, float* __restrict__ part, const int64_t tile, const int N,
                                               const int bn0, const int tid) {
  for (int i = tid; i < BN; i += 512) {
    if (bn0 + i >= N) break;
    float s = 0.f, qv = 0.f;
#pragma unroll
    for (int w = 0; w < WGM; ++w) { s += table[(w * BN + i) * 2]; qv += table[(w * BN + i) * 2 + 1]; }
    part[(tile * 2) * N + bn0 + i] = s;
    part[(tile * 2 + 1) * N + bn0 + i] = qv;
  }
}

}  // namespace
