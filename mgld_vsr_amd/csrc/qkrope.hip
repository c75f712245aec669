// qkrope.hip — root-mean-square norm of every query / key head and the position rotation, one pass over the two projections, and its gradient.
//
//   n = x r g,  r = (mean_d x^2 + eps)^-1/2;   pair (a, b) of n at position p:  (a cos - b sin, a sin + b cos),  angle = p freqs[j]
//   gradient: z = R^T dy,  dg = sum_{rows, heads} z x r,  dx = r (g z - x r mean_d(g z x r))
//
// Bound: HBM (forward 4 bytes per element, gradient 6; 16384 tokens x 40 heads x 128: 67 us, 5.0 TB/s, and 90 us, 5.6 TB/s, where a
// large copy reaches 5.1); everything a head needs sits in the registers of one group of lanes.
//  * A lane holds P = 8 pairs (two 16-byte loads; P = 4 / 8-byte loads where sizes or alignment ask for it), a head is a group of
//    d / 2P lanes padded to a power of two, so the sum of squares is log2(group) exchanges and no LDS.
//  * The sines of a block's tokens are computed once, one pair per thread, and pass through LDS; a group keeps ONE token and walks over heads with
//    its P sines and cosines in registers.  (Every group for itself: 96 us on 16384 tokens x 40 heads x 128, the redundant sincospi held
//    the VALU.)  The angle is reduced in fp64 (turns = p * freqs / 2 pi minus its nearest integer: 2^-31 of a turn at p = 2^20, where an
//    fp32 product is off by 2^-4), then sincospi in fp32.
//  * The gammas lie in LDS (84 vector registers instead of 110: five waves per SIMD, 83 -> 71 us), two heads are in flight per group (-> 70 us),
//    and the results are stored past the L2 (-> 67 us; a reader right behind it does not lose: 129 -> 122 us with a copy of q following,
//    25.1 -> 25.4 us where all of it would fit the caches).
//  * dg is summed in fp32 inside a block (a lane over its tokens and heads, then the groups in order) and in fp64 over the blocks, in a
//    fixed order: the same call gives the same bits.
#include "common.h"

namespace {

typedef __bf16 bf16;
template <typename T, int N> struct qr_vec { typedef T type __attribute__((ext_vector_type(N))); };

// P pairs of a head as this lane holds them: (a[i], b[i]); element indices of the two halves it loads
template <int P, bool IL>
struct PairMap {
  int e0, e1;        // first element of the lane's two P-element vectors
  bool rot, on;
  int j0;            // first pair (index into freqs) when rot
  __device__ PairMap(const int slot, const int d, const int rd) {
    const int p = slot * P;
    on = 2 * p < d;
    rot = 2 * p < rd;
    j0 = p;
    if (IL) { e0 = 2 * p; e1 = 2 * p + P; }
    else if (rot) { e0 = p; e1 = rd / 2 + p; }
    else { e0 = rd + (p - rd / 2); e1 = e0 + (d - rd) / 2; }
  }
};

template <typename T, int P>
struct Raw {               // a lane's two vectors as loaded
  typename qr_vec<T, P>::type u, v;
};
template <typename T, int P, bool IL>
__device__ __forceinline__ void fetch(const T* x, const PairMap<P, IL>& m, Raw<T, P>& r) {
  r.u = *(const typename qr_vec<T, P>::type*)(x + m.e0);
  r.v = *(const typename qr_vec<T, P>::type*)(x + m.e1);
}
template <typename T, int P, bool IL>
__device__ __forceinline__ void unpack(const Raw<T, P>& r, const bool on, float (&a)[P], float (&b)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (IL) {
      a[i] = (float)(2 * i < P ? r.u[(2 * i) % P] : r.v[(2 * i) % P]);
      b[i] = (float)(2 * i < P ? r.u[(2 * i + 1) % P] : r.v[(2 * i + 1) % P]);
    } else {
      a[i] = (float)r.u[i];
      b[i] = (float)r.v[i];
    }
    a[i] = on ? a[i] : 0.f;
    b[i] = on ? b[i] : 0.f;
  }
}
template <typename T, int P, bool IL>
__device__ __forceinline__ void store_pairs(T* y, const PairMap<P, IL>& m, const float (&a)[P], const float (&b)[P]) {
  typedef typename qr_vec<T, P>::type V;
  V u, v;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    if (IL) {
      if (2 * i < P) { u[(2 * i) % P] = (T)a[i]; u[(2 * i + 1) % P] = (T)b[i]; }
      else { v[(2 * i) % P] = (T)a[i]; v[(2 * i + 1) % P] = (T)b[i]; }
    } else {
      u[i] = (T)a[i];
      v[i] = (T)b[i];
    }
  }
  __builtin_nontemporal_store(u, (V*)(y + m.e0));
  __builtin_nontemporal_store(v, (V*)(y + m.e1));
}
template <int P, bool IL>
__device__ __forceinline__ void load_gamma(const float* g, const PairMap<P, IL>& m, float (&a)[P], float (&b)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int ea = IL ? m.e0 + 2 * i : m.e0 + i, eb = IL ? m.e0 + 2 * i + 1 : m.e1 + i;
    a[i] = g && m.on ? g[ea] : 1.f;
    b[i] = g && m.on ? g[eb] : 1.f;
  }
}
// cosine and sine of the rot_dim / 2 pairs of tokens [row0, row0 + n) -> sc[token][pair]; all 256 threads
__device__ __forceinline__ void turns_to_lds(const MgldQkRope& p, const int64_t row0, const int n, f32x2* sc) {
  const int np = p.rot_dim / 2;
  for (int x = threadIdx.x; x < n * np; x += 256) {
    const int tok = x / np, j = x - tok * np;
    const int64_t row = row0 + tok;
    if (row >= p.rows) break;
    const double pos = p.pos64 ? (double)((const int64_t*)p.pos)[row] : (double)((const int32_t*)p.pos)[row];
    double t = pos * (p.freqs[j] * 0.15915494309189533577);
    t -= rint(t);
    float s, c;
    sincospif(2.f * (float)t, &s, &c);
    sc[x] = f32x2{c, s};
  }
}
template <int P, bool IL>
__device__ __forceinline__ void lane_turns(const f32x2* sc, const PairMap<P, IL>& m, float (&c)[P], float (&s)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const f32x2 v = m.on && m.rot ? sc[m.j0 + i] : f32x2{1.f, 0.f};
    c[i] = v[0];
    s[i] = v[1];
  }
}
template <int LG>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// one block: TB = 256 / (LG * GT) tokens, GT groups per token; a group takes heads h = its index, + GT, ...
template <typename T, int P, int LG, bool IL>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const MgldQkRope p, const int GT) {
  extern __shared__ __attribute__((aligned(16))) f32x2 sturn[];    // [TB][rot_dim / 2], then the two gammas
  const int grp = threadIdx.x / LG, slot = threadIdx.x % LG, TB = 256 / LG / GT;
  float* const sgam = (float*)(sturn + TB * (p.rot_dim / 2));
  const int64_t row0 = (int64_t)blockIdx.x * TB, row = row0 + grp / GT;
  const PairMap<P, IL> m(slot, p.head_dim, p.rot_dim);
  const float inv_d = 1.f / (float)p.head_dim;
  const int first = (int)blockIdx.y * GT + grp % GT, step = GT * (int)gridDim.y, H = p.q.heads + p.k.heads;
  auto src = [&](const int h) __attribute__((always_inline)) {
    return h < p.q.heads ? (const T*)p.q.x + row * p.q.x_sr + (int64_t)h * p.q.x_sh
                         : (const T*)p.k.x + row * p.k.x_sr + (int64_t)(h - p.q.heads) * p.k.x_sh;
  };
  float c[P], s[P];
  Raw<T, P> cur, nxt, nx2;
  if (row < p.rows && first < H && m.on) fetch<T, P, IL>(src(first), m, cur);
  if (row < p.rows && first + step < H && m.on) fetch<T, P, IL>(src(first + step), m, nxt);
  turns_to_lds(p, row0, TB, sturn);
  for (int x = threadIdx.x; x < 2 * p.head_dim; x += 256) {
    const bool q = x < p.head_dim;
    const float* g = q ? p.q.gamma : p.k.gamma;
    sgam[x] = g ? g[q ? x : x - p.head_dim] : 1.f;
  }
  __syncthreads();
  if (row >= p.rows) return;
  lane_turns<P, IL>(sturn + (grp / GT) * (p.rot_dim / 2), m, c, s);
  for (int h = first; h < H; h += step) {
    if (h + 2 * step < H && m.on) fetch<T, P, IL>(src(h + 2 * step), m, nx2); // two heads are on their way while this one is turned
    float a[P], b[P];
    unpack<T, P, IL>(cur, m.on, a, b);
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) sq += a[i] * a[i] + b[i] * b[i];
    const float r = rsqrtf(group_sum<LG>(sq) * inv_d + p.eps);
    const bool isq = h < p.q.heads;
    if (m.on) {
      float ya[P], yb[P], ga[P], gb[P];
      load_gamma<P, IL>(sgam + (isq ? 0 : p.head_dim), m, ga, gb);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float u = a[i] * r * ga[i], v = b[i] * r * gb[i];
        ya[i] = u * c[i] - v * s[i];
        yb[i] = u * s[i] + v * c[i];
      }
      T* y = isq ? (T*)p.q.y + row * p.q.y_sr + (int64_t)h * p.q.y_sh : (T*)p.k.y + row * p.k.y_sr + (int64_t)(h - p.q.heads) * p.k.y_sh;
      store_pairs<T, P, IL>(y, m, ya, yb);
    }
    cur = nxt;
    nxt = nx2;
  }
}

// gradient: blocks walk over chunks of QR_CHUNK tokens; one side (queries or keys) per blockIdx.y, so a lane sums one gamma gradient.  A group takes
// (token, head) items in turn, the next one's rows on their way.
constexpr int QR_CHUNK = 8;
template <typename T, int P, int LG, bool IL>
__global__ __launch_bounds__(256) void qk_norm_rope_grad_kernel(const MgldQkRope p) {
  extern __shared__ __attribute__((aligned(16))) float sg[];       // [QR_CHUNK][rot_dim / 2] turns, later [groups][head_dim] gamma sums
  const MgldHeads& sd = blockIdx.y ? p.k : p.q;
  const int grp = threadIdx.x / LG, slot = threadIdx.x % LG, d = p.head_dim;
  constexpr int NG = 256 / LG;
  const PairMap<P, IL> m(slot, d, p.rot_dim);
  const float inv_d = 1.f / (float)d;
  const int H = (int)sd.heads;
  float ga[P], gb[P], da[P], db[P];
  load_gamma<P, IL>(sd.gamma, m, ga, gb);
#pragma unroll
  for (int i = 0; i < P; ++i) { da[i] = 0.f; db[i] = 0.f; }
  for (int64_t row0 = (int64_t)blockIdx.x * QR_CHUNK; row0 < p.rows; row0 += (int64_t)gridDim.x * QR_CHUNK) {
    const int nt = (int)(p.rows - row0 < QR_CHUNK ? p.rows - row0 : QR_CHUNK), items = nt * H;
    Raw<T, P> cx, cg, nx, ng;
    auto fetch2 = [&](const int it, Raw<T, P>& x, Raw<T, P>& g) __attribute__((always_inline)) {
      const int64_t row = row0 + it / H;
      const int h = it % H;
      fetch<T, P, IL>((const T*)sd.x + row * sd.x_sr + (int64_t)h * sd.x_sh, m, x);
      fetch<T, P, IL>((const T*)sd.dy + row * sd.dy_sr + (int64_t)h * sd.dy_sh, m, g);
    };
    if (grp < items && m.on) fetch2(grp, cx, cg);
    __syncthreads();                                               // the previous chunk's turns are used up
    turns_to_lds(p, row0, nt, (f32x2*)sg);
    __syncthreads();
    for (int it = grp; it < items; it += NG) {
      const int64_t row = row0 + it / H;
      const int h = it % H;
      if (it + NG < items && m.on) fetch2(it + NG, nx, ng);
      float c[P], s[P], a[P], b[P], ua[P], ub[P];
      unpack<T, P, IL>(cx, m.on, a, b);
      unpack<T, P, IL>(cg, m.on, ua, ub);
      lane_turns<P, IL>((const f32x2*)sg + (it / H) * (p.rot_dim / 2), m, c, s);
      float sq = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float za = ua[i] * c[i] + ub[i] * s[i], zb = ub[i] * c[i] - ua[i] * s[i];
        ua[i] = za;
        ub[i] = zb;
        sq += a[i] * a[i] + b[i] * b[i];
        dot += za * ga[i] * a[i] + zb * gb[i] * b[i];
      }
      const float r = rsqrtf(group_sum<LG>(sq) * inv_d + p.eps);
      dot = group_sum<LG>(dot) * r * inv_d;                          // mean_d(g z x r)
      if (m.on) {
        float ya[P], yb[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float xa = a[i] * r, xb = b[i] * r;
          da[i] += ua[i] * xa;
          db[i] += ub[i] * xb;
          ya[i] = r * (ua[i] * ga[i] - xa * dot);
          yb[i] = r * (ub[i] * gb[i] - xb * dot);
        }
        store_pairs<T, P, IL>((T*)sd.y + row * sd.y_sr + (int64_t)h * sd.y_sh, m, ya, yb);
      }
      cx = nx;
      cg = ng;
    }
  }
  __syncthreads();
  if (!sd.dgamma) return;
  if (m.on) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int ea = IL ? m.e0 + 2 * i : m.e0 + i, eb = IL ? m.e0 + 2 * i + 1 : m.e1 + i;
      sg[grp * d + ea] = da[i];
      sg[grp * d + eb] = db[i];
    }
  }
  __syncthreads();
  float* out = p.work + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * d;
  for (int e = threadIdx.x; e < d; e += 256) {
    float t = 0.f;
    for (int g = 0; g < NG; ++g) t += sg[g * d + e];
    out[e] = t;
  }
}

// dgamma[e] = sum over the blocks' partial rows, fp64, fixed order: 8 columns x 128 segments of blocks per block (a wave reads 8 rows of 32 bytes;
// 16 columns x 16 segments took 17 us for 1024 rows: one load after the other)
__global__ __launch_bounds__(1024) void qk_gamma_sum_kernel(const MgldQkRope p, const int nblk) {
  __shared__ double sd[128][9];
  float* out = blockIdx.y ? p.k.dgamma : p.q.dgamma;
  if (!out) return;
  const int col = threadIdx.x & 7, seg = threadIdx.x >> 3, e = blockIdx.x * 8 + col;      // head_dim is a multiple of 8
  double t = 0.;
#pragma unroll 4
  for (int i = seg; i < nblk; i += 128) t += (double)p.work[((int64_t)blockIdx.y * nblk + i) * p.head_dim + e];
  sd[seg][col] = t;
  __syncthreads();
  for (int o = 64; o > 0; o >>= 1) {
    if (seg < o) sd[seg][col] += sd[seg + o][col];
    __syncthreads();
  }
  if (seg == 0) out[e] = (float)sd[0][col];
}

// of the gradient, per side (partial gamma rows): four blocks per CU are resident, and every block gets the same number of chunks.  1024 blocks: 95 | 30 us
// (16384 tokens x 40 heads x 128 | 8195 x 32 x 64), 512 in equal shares: 90 | 26, 2048: 102 | 30; chunks of 4 tokens 98 | 40.
constexpr int QR_MAX_BLOCKS = 512;

// pairs a lane holds: 8 when sizes and addresses allow 16-byte vectors, else 4, else 0 (refused)
int qr_pairs(const MgldQkRope* p, const bool grad) {
  for (int P = 8; P >= 4; P /= 2) {
    const int64_t bytes = 2 * P;
    bool ok = p->head_dim % (2 * P) == 0 && p->rot_dim % (2 * P) == 0;
    for (int i = 0; i < 2; ++i) {
      const MgldHeads& h = i ? p->k : p->q;
      if (!h.heads) continue;
      ok = ok && ((uintptr_t)h.x | (uintptr_t)h.y) % bytes == 0 && h.x_sr % P == 0 && h.x_sh % P == 0 && h.y_sr % P == 0 && h.y_sh % P == 0;
      if (grad) ok = ok && (uintptr_t)h.dy % bytes == 0 && h.dy_sr % P == 0 && h.dy_sh % P == 0;
    }
    if (ok) return P;
  }
  return 0;
}

int qr_check(const MgldQkRope* p, const bool grad) {
  MGLD_REQUIRE(p && p->rows >= 0 && p->rows <= 0x7fffffff, "qk_norm_rope: rows");
  MGLD_REQUIRE(p->head_dim >= 8 && p->head_dim <= 256 && p->head_dim % 8 == 0, "qk_norm_rope: head_dim must be a multiple of 8 up to 256");
  MGLD_REQUIRE(p->rot_dim >= 0 && p->rot_dim <= p->head_dim && p->rot_dim % 8 == 0, "qk_norm_rope: rot_dim must be a multiple of 8 up to head_dim");
  MGLD_REQUIRE(p->q.heads >= 0 && p->k.heads >= 0 && p->q.heads + p->k.heads > 0 && p->q.heads <= 65535 && p->k.heads <= 65535, "qk_norm_rope: heads");
  MGLD_REQUIRE(p->eps >= 0.f, "qk_norm_rope: eps");
  if (p->rows == 0) return MGLD_OK;
  MGLD_REQUIRE(p->rot_dim == 0 || (p->pos && p->freqs), "qk_norm_rope: pos / freqs");
  for (int i = 0; i < 2; ++i) {
    const MgldHeads& h = i ? p->k : p->q;
    MGLD_REQUIRE(!h.heads || (h.x && h.y && (!grad || h.dy)), "qk_norm_rope: null pointer");
  }
  MGLD_REQUIRE(qr_pairs(p, grad) > 0, "qk_norm_rope: pointers and strides must be multiples of 8 bytes");
  return MGLD_OK;
}

int qr_grad_blocks(const int64_t rows) {
  const int64_t n = (rows + QR_CHUNK - 1) / QR_CHUNK, turns = (n + QR_MAX_BLOCKS - 1) / QR_MAX_BLOCKS;
  return (int)((n + turns - 1) / turns);
}

template <typename T, int P, int LG, bool IL>
int qr_launch(const MgldQkRope& p, const bool grad, hipStream_t st) {
  constexpr int NG = 256 / LG;
  if (!grad) {
    // many rows: a group walks several heads of its token (sines once per token); few rows: one head per group, heads over blockIdx.y.  Few | many, us:
    // 40 heads of 128 bf16: 256 rows 4.5 | 7.6, 1024 9.4 | 9.3, 2048 15.2 | 10.9, 4096 27.5 | 19.3, 16384 86 | 53;  32 of 64 fp16: 2048 6.7 | 8.2, 3000 9.3 | 9.0, 4096 10.7 | 9.6;
    // 10 of 64: 2048 4.7 | 8.4, 4096 6.4 | 9.5, 6000 8.9 | 9.7, 8192 10.2 | 10.0.  4096 lies between the crossings (1000 .. 8000, by the heads).
    const int H = p.q.heads + p.k.heads;
    int GT = NG;
    if (p.rows >= 4096) while (GT > 1 && GT * 4 > H) GT /= 2;
    else while (GT > 1 && GT / 2 >= H) GT /= 2;
    const int gy = p.rows >= 4096 ? 1 : cdiv(H, GT);
    const int TB = NG / GT;
    qk_norm_rope_kernel<T, P, LG, IL><<<dim3(cdiv(p.rows, TB), gy), 256, (TB * p.rot_dim + 2 * p.head_dim) * 4, st>>>(p, GT);
    return mgld_check_launch("qk_norm_rope");
  }
  const int nb = qr_grad_blocks(p.rows);
  const int lds = (NG * p.head_dim > QR_CHUNK * p.rot_dim ? NG * p.head_dim : QR_CHUNK * p.rot_dim) * 4;
  qk_norm_rope_grad_kernel<T, P, LG, IL><<<dim3(nb, 2), 256, lds, st>>>(p);
  if (p.q.dgamma || p.k.dgamma) qk_gamma_sum_kernel<<<dim3(p.head_dim / 8, 2), 1024, 0, st>>>(p, nb);
  return mgld_check_launch("qk_norm_rope_grad");
}

template <typename T, int P, bool IL>
int qr_lanes(const MgldQkRope& p, const bool grad, hipStream_t st) {
  const int lanes = cdiv(p.head_dim, 2 * P);
  if (lanes <= 4) return qr_launch<T, P, 4, IL>(p, grad, st);
  if (lanes <= 8) return qr_launch<T, P, 8, IL>(p, grad, st);
  if (lanes <= 16) return qr_launch<T, P, 16, IL>(p, grad, st);
  return qr_launch<T, P, 32, IL>(p, grad, st);
}
template <typename T, int P>
int qr_layout(const MgldQkRope& p, const bool grad, hipStream_t st) {
  return p.interleaved ? qr_lanes<T, P, true>(p, grad, st) : qr_lanes<T, P, false>(p, grad, st);
}
int qr_run(const MgldQkRope& p, const bool grad, hipStream_t st) {
  const bool wide = qr_pairs(&p, grad) == 8;
  if (p.bf16) return wide ? qr_layout<bf16, 8>(p, grad, st) : qr_layout<bf16, 4>(p, grad, st);
  return wide ? qr_layout<f16, 8>(p, grad, st) : qr_layout<f16, 4>(p, grad, st);
}

}  // namespace

extern "C" int mgld_qk_norm_rope(const MgldQkRope* p, void* stream) {
  const int rc = qr_check(p, false);
  if (rc || p->rows == 0) return rc;
  return qr_run(*p, false, (hipStream_t)stream);
}

extern "C" int64_t mgld_qk_norm_rope_grad_work(const MgldQkRope* p) {
  if (!p || p->rows <= 0) return 0;
  return (int64_t)2 * qr_grad_blocks(p->rows) * p->head_dim * 4;
}

extern "C" int mgld_qk_norm_rope_grad(const MgldQkRope* p, void* stream) {
  const int rc = qr_check(p, true);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (p->rows == 0) {          // no rows: the sums over them are zero
    if (p->q.dgamma || p->k.dgamma) qk_gamma_sum_kernel<<<dim3(p->head_dim / 8, 2), 1024, 0, st>>>(*p, 0);
    return mgld_check_launch("qk_norm_rope_grad");
  }
  if (p->q.dgamma || p->k.dgamma)
    MGLD_REQUIRE(p->work && p->work_bytes >= mgld_qk_norm_rope_grad_work(p) && (uintptr_t)p->work % 16 == 0, "qk_norm_rope_grad: work buffer too small");
  return qr_run(*p, true, st);
}
