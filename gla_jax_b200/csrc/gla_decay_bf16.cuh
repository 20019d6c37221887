// The walks of gla_decay.cuh for bf16 and head sizes up to 128, which bound by the tensor cores: four warps with 32 (16)
// value columns each, two blocks per SM, the next chunk requested while this one is multiplied; and a backward walk that
// makes dk, dv, the gate's gradient and the first state's gradient together.
//
// Why 32 columns a warp.  Every warp loads the whole of Q and K as fragments; with 16 columns those loads, not the products,
// set the pace (3800 cycles of shared memory against 2700 of mma.sync per 64 tokens at 128 x 128), with 32 they take 2100.
// Why two planes of the weighted values.  The state as an operand is rounded to bf16 anyway; with the weighted values rounded
// to bf16 as well an output is off by sqrt(3) roundings of its own size, with two planes (2^-17) by sqrt(2).
//
// Tiles lie in shared memory without padding, the 16-byte pieces of row r at piece ^ (r % 8), so that two stages of three
// tiles fit twice on an SM and the eight rows of a matrix load fall into different banks.
#pragma once
#include <type_traits>
#include "gla_decay.cuh"

namespace gla {
namespace decay {

template <int PITCH> __device__ __forceinline__ uint32_t at16(uint32_t base, int r, int piece) {      // PITCH bytes a row
  return base + r * PITCH + ((piece ^ (r & 7)) << 4);
}
// Matrix loads of 16 x 16 at (row, column) of a tile, both multiples of 16: lane offsets of the two patterns, to which the
// column is added by exclusive or and the row as it is.  lane_a: A [m][k] (ldsm), B [k][n] (ldsm_t); lane_b: A [k][m]
// (ldsm_t), B [n][k] (ldsm).
template <int PITCH> __device__ __forceinline__ uint32_t lane_a(int lane) { return (lane & 15) * PITCH + (((lane >> 4) ^ (lane & 7)) << 4); }
template <int PITCH> __device__ __forceinline__ uint32_t lane_b(int lane) {
  return ((lane & 7) + ((lane >> 4) & 1) * 8) * PITCH + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
}
// A chunk of 64 rows into a tile: a thread's 16-byte pieces lie NT / (D / 8) rows apart.  src: row 0 of the chunk.
template <int D, int NT>
__device__ __forceinline__ void fetch_tile(uint32_t tile, const bf16* src, int64_t step, int nv, int d) {
  constexpr int C8 = D / 8, RS = NT / C8;
  static_assert(RS % 8 == 0, "the pieces of a thread lie at one place of their rows");
  const int r0 = threadIdx.x / C8, c = threadIdx.x % C8;
  const bf16* g = src + r0 * step + c * 8;
  const uint32_t dst = at16<2 * D>(tile, r0, c);
  const int n = c * 8 < d ? nv - r0 : 0;
#pragma unroll
  for (int j = 0; j < 64 / RS; ++j) {
    cp16(dst + j * RS * 2 * D, RS * j < n ? g : src, RS * j < n);
    g += RS * step;
  }
}
__device__ __forceinline__ float ex2(float x) {      // 2^-22 relative, 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// an A fragment times a weight per k (w[0], w[1]: k 2 tq, 2 tq + 1; w[2], w[3]: eight further), in NU planes
template <int NU>
__device__ __forceinline__ void weighted(uint32_t (&z)[NU][4], const uint32_t (&a)[4], const float (&w)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 x = pair_of(a[e]);
    uint32_t s[NU];
    planes<NU>(x.x * w[e / 2 * 2], x.y * w[e / 2 * 2 + 1], s);
#pragma unroll
    for (int i = 0; i < NU; ++i) z[i][e] = s[i];
  }
}

// What a chunk of 64 needs of its gates, made by one warp, two rows a lane.  lam: running sums, base 2, as two floats;
// wt: exp(lam_i) and exp(lam_L - lam_i).  The weight exp(lam_i - lam_j) of a score below the diagonal blocks of 16 x 16 is a
// product rf_i cf_j over the last token before i's block, so that 160 exponentials make 1536 weights.
struct Gates {
  float2 lam[64], wt[64];
  float rf[64], cf[3][64];           // cf[b - 1]: to the last token before row block b
};
__device__ __forceinline__ float2 gates_of(const Walk& p, int64_t t0, int nv, int h, int lane) {
  float2 g = make_float2(0.f, 0.f);
  if (2 * lane < nv) g.x = p.g[(t0 + 2 * lane) * p.gt + h];
  if (2 * lane + 1 < nv) g.y = p.g[(t0 + 2 * lane + 1) * p.gt + h];
  return g;
}
__device__ __forceinline__ double scan_gates(float2 g, Gates& s, int lane) {
  // exp of less than -200 is 0 either way; -inf would leave inf - inf
  const double a = (double)(g.x < -200.f ? -200.f : g.x) * 1.4426950408889634, b = (double)(g.y < -200.f ? -200.f : g.y) * 1.4426950408889634;
  double inc = a + b;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  const double all = __shfl_sync(0xffffffffu, inc, 31), own = __shfl_sync(0xffffffffu, inc, lane >= 8 ? lane / 8 * 8 - 1 : 0);
  const double at[3] = {__shfl_sync(0xffffffffu, inc, 7), __shfl_sync(0xffffffffu, inc, 15), __shfl_sync(0xffffffffu, inc, 23)};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double v = i ? inc : inc - b;
    const float hi = (float)v;
    const int r = 2 * lane + i;
    s.lam[r] = make_float2(hi, (float)(v - hi));
    s.wt[r] = make_float2(ex2(hi), ex2((float)(all - v)));
    s.rf[r] = ex2((float)(v - own));
#pragma unroll
    for (int m = 0; m < 3; ++m)
      if (lane < 8 * (m + 1)) s.cf[m][r] = ex2((float)(at[m] - v));
  }
  return all;
}
__device__ __forceinline__ float decay_of(float2 i, float2 j) { return ex2((i.x - j.x) + (i.y - j.y)); }
// the weights of rows r, r + 8 (index / 2) and columns j, j + 1 of a block
__device__ __forceinline__ void weights_of(float (&w)[4], const Gates& s, int mi, int nj, int r, int j) {
  if (mi == nj) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = r + 8 * (e / 2), c = j + e % 2;
      w[e] = c <= i ? decay_of(s.lam[i], s.lam[c]) : 0.f;
    }
  } else {
    const float2 c = *reinterpret_cast<const float2*>(&s.cf[mi - 1][j]);
    const float a = s.rf[r], b = s.rf[r + 8];
    w[0] = a * c.x; w[1] = a * c.y; w[2] = b * c.x; w[3] = b * c.y;
  }
}
// Whether a B fragment holds something that is not finite.  In a diagonal block it would meet the zeros of later (backwards:
// earlier) tokens in the product, and 0 x inf is not a number; the recurrence has it at its own token and after only.
__device__ __forceinline__ bool not_finite(const uint32_t (&b)[4]) {
  bool x = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) x = x || (b[i] & 0x7f80u) == 0x7f80u || (b[i] & 0x7f800000u) == 0x7f800000u;
  return x;
}
__device__ __forceinline__ float lds_bf16(uint32_t a) {
  uint16_t u;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(a));
  return __uint_as_float((uint32_t)u << 16);
}
// Such a block by the sums themselves: o (rows gr, gr + 8 of the block at r0, tiles of 8 columns from c0) += P V over the block's
// own tokens, j <= i; UP: P^T V, over j >= i.
template <int PITCH, int NT8, bool UP>
__device__ __noinline__ void diagonal_sums(float (&o)[NT8][4], uint32_t tp, uint32_t tv, int r0, int c0, int gr, int tq) {
#pragma unroll 1
  for (int j = 0; j < 16; ++j) {
    const int t = r0 + j;
    float s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) s[u] = UP ? lds_bf16(at16<128>(tp, t, (r0 + gr + 8 * u) / 8) + gr * 2) : lds_bf16(at16<128>(tp, r0 + gr + 8 * u, t / 8) + t % 8 * 2);
#pragma unroll
    for (int n = 0; n < NT8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = gr + 8 * (e / 2), c = c0 + 8 * n + 2 * tq + e % 2;
        if (UP ? j >= i : j <= i) o[n][e] = fmaf(s[e / 2], lds_bf16(at16<PITCH>(tv, t, c / 8) + c % 8 * 2), o[n][e]);
      }
  }
}
template <int PITCH, int NT8, bool UP>
__device__ __forceinline__ void diagonal_by_sums(float (&o)[NT8][4], uint32_t tp, uint32_t tv, int r0, int c0, int gr, int tq) {
  float x[NT8][4];                   // (a copy, so that o itself stays in registers)
#pragma unroll
  for (int n = 0; n < NT8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[n][e] = o[n][e];
  diagonal_sums<PITCH, NT8, UP>(x, tp, tv, r0, c0, gr, tq);
#pragma unroll
  for (int n = 0; n < NT8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = x[n][e];
}
// 4 x 4 words across the four lanes of a row: lane tq is left with word tq of each
__device__ __forceinline__ void transpose4(uint32_t (&v)[4], int tq) {
#pragma unroll
  for (int s = 1; s < 4; s <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (!(j & s)) {
        const uint32_t y = __shfl_xor_sync(0xffffffffu, (tq & s) ? v[j] : v[j | s], s);
        if (tq & s) v[j] = y; else v[j | s] = y;
      }
}

template <int KD, int NC, bool OUT>
struct FLay {
  static constexpr int VT = 64 * NC, NT = 128;
  static constexpr int PK = 128 * KD, PV = 128 * VT, STAGE = (OUT ? 2 : 1) * PK + PV;
  static constexpr int P0 = 2 * STAGE, G0 = P0 + (OUT ? 8192 : 0), RD = G0 + 2 * (int)sizeof(Gates), END = RD + (OUT ? 1024 : 0);
};

// KD: features; NC: groups of 16 value columns of a warp; NU: planes of the weighted values (3: and exact additions); NS:
// planes of the state as an operand
template <int KD, int NC, int NU, int NS, bool OUT>
__global__ void __launch_bounds__(128, 2) fast_walk_kernel(const Walk p) {
  using Y = FLay<KD, NC, OUT>;
  constexpr int KT = KD / 8, QP = 2 * KD, VP = 2 * Y::VT;
  extern __shared__ __align__(256) uint8_t sm[];
  Gates* gates = reinterpret_cast<Gates*>(sm + Y::G0);
  float* rd = reinterpret_cast<float*>(sm + Y::RD);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, gr = lane / 4, tq = lane % 4;
  const int h = blockIdx.y % p.H, vt = blockIdx.y / p.H;
  const int cbase = vt * Y::VT, cl = warp * 16 * NC, cw = cbase + cl;
  const Run run = find_run(p, blockIdx.x);
  if constexpr (OUT) {
    if (run.zlo < run.zhi) {
      const int w = p.vd - cbase < Y::VT ? p.vd - cbase : Y::VT;
      for (int64_t i = tid; i < (run.zhi - run.zlo) * w; i += Y::NT)
        st_any(p.out, !p.out_f32, ((run.zlo + i / w) * p.H + h) * p.vd + cbase + i % w, 0.f);
    }
    if (p.count_bad && run.any && run.first && blockIdx.y == 0 && tid == 0) {
      const int64_t a = p.cu ? p.cu[run.s] : 0, b = p.cu ? p.cu[run.s + 1] : 0;
      if (p.cu && (a < 0 || b < a || b > p.T || (run.s == 0 && a != 0))) atomicAdd(&g_bad_offsets, 1u);
    }
  }
  if (!run.any) return;
  if (!OUT && (p.rev ? run.first : run.last)) return;

  const int64_t sh = run.s * p.H + h, dd = (int64_t)p.kd * p.vd, slot_h = (int64_t)blockIdx.x * p.H + h;
  const int Hq = p.H / p.gq, Hk = p.H / p.gk, Hv = p.H / p.gv;
  const int len = (int)(run.hi - run.lo), chunks = (len + 63) / 64;
  const uint32_t base = sm32(sm);
  const int64_t r0 = run.base + run.lo;                                   // the run's first token
  const int64_t sk = (int64_t)Hk * p.kd, sv = (int64_t)Hv * p.vd, sq = (int64_t)Hq * p.kd;
  const bf16* gk = (const bf16*)p.k + r0 * sk + h / p.gk * p.kd;
  const bf16* gv = (const bf16*)p.v + r0 * sv + h / p.gv * p.vd + cbase;
  const bf16* gq = OUT ? (const bf16*)p.q + r0 * sq + h / p.gq * p.kd : nullptr;
  // chunk i of the walk; backwards in time (sums only) from the last one
  const auto first_of = [&](int i) { return 64 * (p.rev ? chunks - 1 - i : i); };
  const auto fetch = [&](int i) {
    const int c0 = first_of(i), nv = len - c0 < 64 ? len - c0 : 64;
    const uint32_t s = base + (i & 1) * Y::STAGE;
    fetch_tile<KD, 128>(s, gk + c0 * sk, sk, nv, p.kd);
    fetch_tile<Y::VT, 128>(s + Y::PK, gv + c0 * sv, sv, nv, p.vd - cbase);
    if constexpr (OUT) fetch_tile<KD, 128>(s + Y::PK + Y::PV, gq + c0 * sq, sq, nv, p.kd);
  };
  double total = 0.0;
  if (chunks) {
    fetch(0);
    if (warp == 0) {
      const int c0 = first_of(0);
      total += scan_gates(gates_of(p, r0 + c0, len - c0 < 64 ? len - c0 : 64, h, lane), gates[0], lane);
    }
  }
  cp_commit();

  float st[NC][KT][4];
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = cw + 16 * n + gr + 8 * (e / 2), k = 8 * j + 2 * tq + e % 2;
        float x = 0.f;
        if (OUT && c < p.vd && k < p.kd)
          x = p.seg_state ? p.seg_state[slot_h * dd + k * p.sk + c * p.sc] : ld_any(p.init, !p.init_f32, sh * dd + k * p.ik + c * p.ic);
        st[n][j][e] = x;
      }

  const uint32_t laq = lane_a<QP>(lane), lbq = lane_b<QP>(lane), lav = lane_a<VP>(lane) ^ (cl * 2), lbv = lane_b<VP>(lane) ^ (cl * 2), lap = lane_a<128>(lane);
  for (int i = 0; i < chunks; ++i) {
    const int c0 = first_of(i), nv = len - c0 < 64 ? len - c0 : 64;
    const int64_t t0 = r0 + c0;
    const uint32_t uk = base + (i & 1) * Y::STAGE, uv = uk + Y::PK, uq = uv + Y::PV, up = base + Y::P0;
    const Gates& gs = gates[i & 1];
    cp_wait<0>();
    __syncthreads();                 // this chunk is here, and nobody reads the other stage any more
    float2 gn = make_float2(0.f, 0.f);
    if (i + 1 < chunks) {
      fetch(i + 1);
      if (warp == 0) {
        const int n0 = first_of(i + 1);
        gn = gates_of(p, r0 + n0, len - n0 < 64 ? len - n0 : 64, h, lane);
      }
    }
    cp_commit();
    if constexpr (OUT) {
      if (p.r && i > 0 && tid < 64)
        // the row sums of the chunk before (a whole one)
        p.rdot[(vt * (p.cu ? p.T : p.nseq * p.T) + t0 - 64 + tid) * p.H + h] = (rd[tid] + rd[64 + tid]) + (rd[128 + tid] + rd[192 + tid]);
      // scores in blocks of 16 x 16: (3,0) (3,1) | (3,2) (3,3) | (2,0) (2,1) (2,2) | (1,0) (1,1) (0,0)
#pragma unroll 1
      for (int b = 0; b < (warp < 2 ? 2 : 3); ++b) {
        const int mi = warp < 2 ? 3 : warp == 2 ? 2 : b < 2 ? 1 : 0, nj = warp == 1 ? 2 + b : warp == 3 && b == 2 ? 0 : b;
        if (mi * 16 >= nv) continue;
        float c[2][4] = {};
        const uint32_t qa = uq + mi * 16 * QP, ka = uk + nj * 16 * QP;
#pragma unroll
        for (int kk = 0; kk < KD / 16; ++kk) {
          uint32_t a[4], x[4];
          ldsm(a, qa + (laq ^ (kk * 32)));
          ldsm(x, ka + (lbq ^ (kk * 32)));
          mma16(c[0], a, x[0], x[1]);
          mma16(c[1], a, x[2], x[3]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int r = mi * 16 + gr, j = nj * 16 + n * 8 + 2 * tq;
          float w[4];
          weights_of(w, gs, mi, nj, r, j);
          // (a score of a masked pair may be anything: 0 by selection)
          const bool d = mi == nj;
#pragma unroll
          for (int e = 0; e < 4; ++e) c[n][e] = d && j + e % 2 > r + 8 * (e / 2) ? 0.f : c[n][e] * w[e];
          const uint32_t at = at16<128>(up, r, 2 * nj + n) + 4 * tq;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(pack_bf16x2(c[n][0], c[n][1])) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + 8 * 128), "r"(pack_bf16x2(c[n][2], c[n][3])) : "memory");
        }
      }
    }
    if (warp == 0 && i + 1 < chunks) total += scan_gates(gn, gates[(i + 1) & 1], lane);
    if constexpr (OUT) {
      __syncthreads();
#pragma unroll 1
      for (int m = 0; m < 64 && m < nv; m += 32) {
          float o[2][2 * NC][4] = {};
#pragma unroll
          for (int kk = 0; kk < KD / 16; ++kk) {
            uint32_t a[2][4];
            ldsm(a[0], uq + m * QP + (laq ^ (kk * 32)));
            ldsm(a[1], uq + (m + 16) * QP + (laq ^ (kk * 32)));
            uint32_t b[NC][4][NS];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
              planes<NS>(st[n][2 * kk][0], st[n][2 * kk][1], b[n][0]);
              planes<NS>(st[n][2 * kk + 1][0], st[n][2 * kk + 1][1], b[n][1]);
              planes<NS>(st[n][2 * kk][2], st[n][2 * kk][3], b[n][2]);
              planes<NS>(st[n][2 * kk + 1][2], st[n][2 * kk + 1][3], b[n][3]);
            }
#pragma unroll
            for (int s = NS - 1; s >= 0; --s)
#pragma unroll
              for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  mma16(o[r][2 * n], a[r], b[n][0][s], b[n][1][s]);
                  mma16(o[r][2 * n + 1], a[r], b[n][2][s], b[n][3][s]);
                }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float w0 = gs.wt[m + 16 * r + gr].x, w1 = gs.wt[m + 16 * r + gr + 8].x;
#pragma unroll
            for (int n = 0; n < 2 * NC; ++n) { o[r][n][0] *= w0; o[r][n][1] *= w0; o[r][n][2] *= w1; o[r][n][3] *= w1; }
          }
          if (p.r) {
            // the rows' products with what comes from before the chunk
            const int Hr = p.H / p.gr;
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int row = m + 16 * r + gr + 8 * half;
                float dot = 0.f;
                if (row < nv) {
                  const int64_t ra = ((t0 + row) * Hr + h / p.gr) * p.vd + cw + 2 * tq;
#pragma unroll
                  for (int n = 0; n < 2 * NC; ++n)
                    if (cw + 8 * n < p.vd) {
                      const float2 x = pair_of(__ldg((const unsigned int*)((const bf16*)p.r + ra + 8 * n)));
                      dot = fmaf(o[r][n][2 * half], x.x, fmaf(o[r][n][2 * half + 1], x.y, dot));
                    }
                }
                dot += __shfl_xor_sync(0xffffffffu, dot, 1);
                dot += __shfl_xor_sync(0xffffffffu, dot, 2);
                if (tq == 0) rd[warp * 64 + row] = dot;
              }
          }
#pragma unroll 1
          for (int kj = 0; kj <= m + 16; kj += 16) {
            uint32_t a[2][4], b[NC][4];
            bool odd = false;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
              ldsm_t(b[n], uv + kj * VP + (lav ^ (n * 32)));
              odd = odd || not_finite(b[n]);
            }
            odd = __any_sync(0xffffffffu, odd);
            ldsm(a[1], up + (m + 16) * 128 + (lap ^ (kj * 2)));
            if (odd && kj == m + 16) {
              diagonal_by_sums<VP, 2 * NC, false>(o[1], up, uv, kj, cl, gr, tq);
            } else {
#pragma unroll
              for (int n = 0; n < NC; ++n) { mma16(o[1][2 * n], a[1], b[n][0], b[n][1]); mma16(o[1][2 * n + 1], a[1], b[n][2], b[n][3]); }
            }
            if (kj <= m) {
              ldsm(a[0], up + m * 128 + (lap ^ (kj * 2)));
              if (odd && kj == m) {
                diagonal_by_sums<VP, 2 * NC, false>(o[0], up, uv, kj, cl, gr, tq);
              } else {
#pragma unroll
                for (int n = 0; n < NC; ++n) { mma16(o[0][2 * n], a[0], b[n][0], b[n][1]); mma16(o[0][2 * n + 1], a[0], b[n][2], b[n][3]); }
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int row = m + 16 * r + gr + 8 * half;
              if (p.out_f32 || NC == 1) {
                const int64_t at = ((t0 + row) * p.H + h) * p.vd + cw + 2 * tq;
#pragma unroll
                for (int n = 0; n < 2 * NC; ++n)
                  if (row < nv && cw + 8 * n < p.vd) {
                    const float x = o[r][n][2 * half], y = o[r][n][2 * half + 1];
                    if (p.out_f32) *reinterpret_cast<float2*>((float*)p.out + at + 8 * n) = make_float2(x, y);
                    else *reinterpret_cast<uint32_t*>((bf16*)p.out + at + 8 * n) = pack_bf16x2(x, y);
                  }
              } else {
                uint32_t v[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) v[n] = pack_bf16x2(o[r][n % (2 * NC)][2 * half], o[r][n % (2 * NC)][2 * half + 1]);
                transpose4(v, tq);
                if (row < nv && cw + 8 * tq < p.vd)
                  *reinterpret_cast<uint4*>((bf16*)p.out + ((t0 + row) * p.H + h) * p.vd + cw + 8 * tq) = make_uint4(v[0], v[1], v[2], v[3]);
              }
            }
      }
    }
    // the state: st = exp(lam_L) st + (w V)^T K, backwards in time with exp(lam_i) as weights
    const float all = gs.wt[63].x;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[n][j][e] *= all;
    const float* ws = &gs.wt[0].x + (p.rev ? 0 : 1);
#pragma unroll 1
    for (int kk = 0; kk < 64 && kk < nv; kk += 16) {
      const int j = 2 * (kk + 2 * tq);
      const float w[4] = {ws[j], ws[j + 2], ws[j + 16], ws[j + 18]};
      uint32_t z[NC][NU][4];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        uint32_t a[4];
        ldsm_t(a, uv + kk * VP + (lbv ^ (n * 32)));
        weighted<NU>(z[n], a, w);
      }
#pragma unroll
      for (int t = 0; t < KD / 16; ++t) {
        uint32_t b[1][4];
        ldsm_t(b[0], uk + kk * QP + (laq ^ (t * 32)));
        if constexpr (NU > 2) {
#pragma unroll
          for (int n = 0; n < NC; ++n) mma_planes<NU, 1, true>(st[n][2 * t], st[n][2 * t + 1], z[n], b);
        } else {
#pragma unroll
          for (int s = NU - 1; s >= 0; --s)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
              mma16(st[n][2 * t], z[n][s], b[0][0], b[0][1]);
              mma16(st[n][2 * t + 1], z[n][s], b[0][2], b[0][3]);
            }
        }
      }
    }
  }

  if constexpr (OUT) {
    if (p.r && chunks) {
      __syncthreads();
      const int c0 = 64 * (chunks - 1);
      if (tid < len - c0)
        p.rdot[(vt * (p.cu ? p.T : p.nseq * p.T) + r0 + c0 + tid) * p.H + h] = (rd[tid] + rd[64 + tid]) + (rd[128 + tid] + rd[192 + tid]);
    }
    if ((p.fin || p.fin32) && run.last) {
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = cw + 16 * n + gr + 8 * (e / 2), k = 8 * j + 2 * tq + e % 2;
            if (c < p.vd && k < p.kd) {
              const int64_t at = sh * dd + k * p.ik + c * p.ic;
              if (p.fin) st_any(p.fin, !p.fin_f32, at, st[n][j][e]);
              if (p.fin32) p.fin32[at] = st[n][j][e];
            }
          }
    }
  } else {
    if (tid == 0 && vt == 0) p.seg_total[slot_h] = total;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int c = cw + 16 * n + gr + 4 * e, k = 8 * j + 2 * tq;
          if (c < p.vd && k < p.kd) *reinterpret_cast<float2*>(p.seg_state + slot_h * dd + (int64_t)c * p.kd + k) = make_float2(st[n][j][e], st[n][j][e + 1]);
        }
  }
}

// ---- backwards: dk, dv, the gates and the first state ----------------------------------------------------------------------
// For a chunk, with dS the gradient of the state that leaves it (P, dP: scores times decay, i >= j):
//   dV = P^T dO + exp(lam_L - lam_j) (K dS)            dK = dP^T Q + exp(lam_L - lam_j) (V dS^T)
//   dS <- exp(lam_L) dS + (exp(lam_i) Q)^T dO
//   e_t = sum_j M_tj - sum_i M_it + a_t - b_t,  M_ij = P_ij (dO_i V_j^T),  a = q . (dq from before the chunk), b = k . (dk from behind it)
//   dg_t = sum of e from t to the run's end + <the state that leaves the run, its gradient>
// M in float32 and the products with states in two planes: the sum is over the whole run and its terms cancel.
// Both products with dS read it from shared memory, one as [k][n], one as [n][k], which is why it is put there each chunk
// and why the update is done once (eight warps, an eighth of dS each) instead of once per orientation in registers.
struct Back {
  Walk w;                                  // k, q, v; H, sizes, gates, runs; seg_state: gradients that enter each run backwards
  const void* dout;
  const float* a;                          // [token][H], with gates
  const float *S_runs, *S_end;             // entering states of the runs [slot][H][vd][kd] (NULL: one run each), final states
  void *dk, *dv;
  int dk_f32;
  float* dg;
};
template <int DK, int DV, int NS>
struct BLay {
  static constexpr int TK = 128 * DK, TV = 128 * DV, STAGE = 2 * TK + 2 * TV;
  static constexpr int S0 = 2 * STAGE, SP = DK * DV * 2, P0 = S0 + NS * SP, D0 = P0 + 8192, G0 = D0 + 8192;
  static constexpr int RS = G0 + 2 * (int)sizeof(Gates), CS = RS + 2 * 2048, BD = CS + 2 * 1024, RED = BD + 2 * 512, END = RED + 64;
};
template <int DK, int DV, bool GATE>
__global__ void __launch_bounds__(256, 1) fast_back_kernel(const Back q) {
  constexpr int NS = GATE ? 2 : 1;
  using Y = BLay<DK, DV, NS>;
  constexpr int KP = 2 * DK, VP = 2 * DV, MR = DK / 64, NV = DV / 16;   // update: MR x 16 rows and NV tiles of 8 columns per warp
  const Walk& p = q.w;
  extern __shared__ __align__(256) uint8_t sm[];
  Gates* gates_ = reinterpret_cast<Gates*>(sm + Y::G0);
  float* rs_ = reinterpret_cast<float*>(sm + Y::RS);           // [2][8 tiles of columns][64]: sums of a row of M over 8 columns
  float* cs_ = reinterpret_cast<float*>(sm + Y::CS);           // [2][4 tiles of rows][64]
  float* bd_ = reinterpret_cast<float*>(sm + Y::BD);           // [2][2 halves][64]
  double* red = reinterpret_cast<double*>(sm + Y::RED);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, gr = lane / 4, tq = lane % 4;
  const int h = blockIdx.y;
  const Run run = find_run(p, blockIdx.x);
  if (run.zlo < run.zhi) {
    for (int64_t i = tid; i < (run.zhi - run.zlo) * p.kd; i += 256) st_any(q.dk, !q.dk_f32, ((run.zlo + i / p.kd) * p.H + h) * p.kd + i % p.kd, 0.f);
    for (int64_t i = tid; i < (run.zhi - run.zlo) * p.vd; i += 256) st_any(q.dv, 1, ((run.zlo + i / p.vd) * p.H + h) * p.vd + i % p.vd, 0.f);
    if (GATE)
      for (int64_t i = tid; i < run.zhi - run.zlo; i += 256) q.dg[(run.zlo + i) * p.H + h] = 0.f;
  }
  if (!run.any) return;
  const int64_t sh = run.s * p.H + h, dd = (int64_t)p.kd * p.vd, slot_h = (int64_t)blockIdx.x * p.H + h;
  const int ur = (warp >> 1) * 16 * MR, uc = (warp & 1) * (DV / 2);       // the warp's part of dS
  float st[MR][NV][4];
  double dot = 0.0;
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = ur + 16 * m + gr + 8 * (e / 2), c = uc + 8 * n + 2 * tq + e % 2;
        float x = 0.f;
        if (c < p.vd && k < p.kd) {
          x = p.seg_state ? p.seg_state[slot_h * dd + (int64_t)c * p.kd + k] : ld_any(p.init, !p.init_f32, sh * dd + k * p.ik + c * p.ic);
          if (GATE) dot += (double)x * (run.last ? q.S_end[sh * dd + (int64_t)k * p.vd + c] : q.S_runs[(slot_h + p.H) * dd + (int64_t)c * p.kd + k]);
        }
        st[m][n][e] = x;
      }
  double carry = 0.0;
  if constexpr (GATE) {
#pragma unroll
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (lane == 0) red[warp] = dot;
    __syncthreads();
    for (int w = 0; w < 8; ++w) carry += red[w];
  }
  const int Hq = p.H / p.gq, len = (int)(run.hi - run.lo), chunks = (len + 63) / 64;
  const uint32_t base = sm32(sm);
  const int64_t r0_ = run.base + run.lo, sk = (int64_t)Hq * p.kd, sv = (int64_t)p.H * p.vd;
  const int64_t ok = r0_ * sk + h / p.gq * p.kd, ov = r0_ * sv + (int64_t)h * p.vd;
  const auto fetch = [&](int i) {
    const int nv = len - 64 * i < 64 ? len - 64 * i : 64;
    const uint32_t s = base + (i & 1) * Y::STAGE;
    const int64_t rk = ok + 64 * i * sk, rv = ov + 64 * i * sv;
    fetch_tile<DK, 256>(s, (const bf16*)p.q + rk, sk, nv, p.kd);
    fetch_tile<DK, 256>(s + Y::TK, (const bf16*)p.k + rk, sk, nv, p.kd);
    fetch_tile<DV, 256>(s + 2 * Y::TK, (const bf16*)p.v + rv, sv, nv, p.vd);
    fetch_tile<DV, 256>(s + 2 * Y::TK + Y::TV, (const bf16*)q.dout + rv, sv, nv, p.vd);
  };
  if (chunks) {
    fetch(chunks - 1);
    if (warp == 0) scan_gates(gates_of(p, r0_ + 64 * (chunks - 1), len - 64 * (chunks - 1), h, lane), gates_[(chunks - 1) & 1], lane);
  }
  cp_commit();
  const uint32_t lak = lane_a<KP>(lane), lbk = lane_b<KP>(lane), lav = lane_a<VP>(lane), lbv = lane_b<VP>(lane), lbp = lane_b<128>(lane);
  // gradient of the gates of chunk i, by one warp, once its sums are there
  const auto gates = [&](int i) {
    const int nv = len - 64 * i < 64 ? len - 64 * i : 64;
    const int64_t t0 = run.base + run.lo + 64 * i;
    const float *rs = rs_ + (i & 1) * 512, *cs = cs_ + (i & 1) * 256, *bd = bd_ + (i & 1) * 128;
    double e[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = 2 * lane + u;
      double x = 0.0;
      if (t < nv) {
        for (int n = 0; n <= t / 16 * 2 + 1; ++n) x += rs[n * 64 + t];
        for (int m = t / 16; m < 4; ++m) x -= cs[m * 64 + t];
        x += (double)q.a[(t0 + t) * p.H + h] - ((double)bd[t] + bd[64 + t]);
      }
      e[u] = x;
    }
    double inc = e[0] + e[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double y = __shfl_down_sync(0xffffffffu, inc, d);
      if (lane + d < 32) inc += y;
    }
    if (2 * lane < nv) q.dg[(t0 + 2 * lane) * p.H + h] = (float)(carry + inc);
    if (2 * lane + 1 < nv) q.dg[(t0 + 2 * lane + 1) * p.H + h] = (float)(carry + inc - e[0]);
    carry += __shfl_sync(0xffffffffu, inc, 0);
  };
  for (int i = chunks - 1; i >= 0; --i) {
    const int nv = len - 64 * i < 64 ? len - 64 * i : 64;
    const int64_t t0 = run.base + run.lo + 64 * i;
    const uint32_t uq = base + (i & 1) * Y::STAGE, uk = uq + Y::TK, uv = uk + Y::TK, uo = uv + Y::TV, us = base + Y::S0, up = base + Y::P0, ud = base + Y::D0;
    const Gates& gs = gates_[i & 1];
    cp_wait<0>();
    __syncthreads();
    float2 gn = make_float2(0.f, 0.f);
    if (i > 0) {
      fetch(i - 1);
      if (warp == 7) gn = gates_of(p, t0 - 64, 64, h, lane);
    }
    cp_commit();
    // dS for the products of this chunk
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int k = ur + 16 * m + gr + 4 * e, c = uc + 8 * n + 2 * tq;
          uint32_t s[NS];
          planes<NS>(st[m][n][e], st[m][n][e + 1], s);
#pragma unroll
          for (int x = 0; x < NS; ++x)
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(at16<VP>(us + x * Y::SP, k, c / 8) + (c % 8) * 2), "r"(s[x]) : "memory");
        }
    // scores and their gradients, 16 x 8 of both at a time
#pragma unroll 1
    for (int u = warp; u < 20; u += 8) {
      const int mi = u < 2 ? 0 : u < 6 ? 1 : u < 12 ? 2 : 3, nt = u - mi * (mi + 1), r = mi * 16 + gr, j = nt * 8 + 2 * tq;
      float c[4] = {}, d[4] = {};
      // eight rows of K (V) x 32 features: four matrices side by side
      const uint32_t l8 = (lane & 7) * KP + (((lane >> 3) ^ (lane & 7)) << 4), l8v = (lane & 7) * VP + (((lane >> 3) ^ (lane & 7)) << 4);
#pragma unroll
      for (int kk = 0; kk < DK / 32; ++kk) {
        uint32_t a[4], a2[4], b[4];
        ldsm(b, uk + nt * 8 * KP + (l8 ^ (kk * 64)));
        ldsm(a, uq + mi * 16 * KP + (lak ^ (kk * 64)));
        ldsm(a2, uq + mi * 16 * KP + (lak ^ (kk * 64 + 32)));
        mma16(c, a, b[0], b[1]);
        mma16(c, a2, b[2], b[3]);
      }
#pragma unroll
      for (int kk = 0; kk < DV / 32; ++kk) {
        uint32_t a[4], a2[4], b[4];
        ldsm(b, uv + nt * 8 * VP + (l8v ^ (kk * 64)));
        ldsm(a, uo + mi * 16 * VP + (lav ^ (kk * 64)));
        ldsm(a2, uo + mi * 16 * VP + (lav ^ (kk * 64 + 32)));
        mma16(d, a, b[0], b[1]);
        mma16(d, a2, b[2], b[3]);
      }
      float w[4], x[4], m[4];
      weights_of(w, gs, mi, nt / 2, r, j);
      const bool diag = mi == nt / 2;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool off = diag && j + e % 2 > r + 8 * (e / 2);
        x[e] = off ? 0.f : c[e] * w[e];
        m[e] = off ? 0.f : x[e] * d[e];
        d[e] = off ? 0.f : d[e] * w[e];
      }
      const uint32_t at = at16<128>(0, r, nt) + 4 * tq;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(up + at), "r"(pack_bf16x2(x[0], x[1])) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(up + at + 1024), "r"(pack_bf16x2(x[2], x[3])) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(ud + at), "r"(pack_bf16x2(d[0], d[1])) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(ud + at + 1024), "r"(pack_bf16x2(d[2], d[3])) : "memory");
      if constexpr (GATE) {
        float a = m[0] + m[1], b = m[2] + m[3], y = m[0] + m[2], z = m[1] + m[3];
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) { a += __shfl_xor_sync(0xffffffffu, a, s); b += __shfl_xor_sync(0xffffffffu, b, s); }
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) { y += __shfl_xor_sync(0xffffffffu, y, s); z += __shfl_xor_sync(0xffffffffu, z, s); }
        float* rs = rs_ + (i & 1) * 512 + nt * 64 + r;
        if (tq == 0) { rs[0] = a; rs[8] = b; }
        if (gr == 0) *reinterpret_cast<float2*>(cs_ + (i & 1) * 256 + mi * 64 + j) = make_float2(y, z);
      }
    }
    if (warp == 7) {
      if (i > 0) scan_gates(gn, gates_[(i - 1) & 1], lane);
      if (GATE && i + 1 < chunks) gates(i + 1);
    }
    __syncthreads();
    // one output's tile of 32 rows (row tiles 0 and 3, or 1 and 2, which have as much before them) x half the columns
    {
      const int r0 = (warp & 1) * 16, r1 = 48 - r0, half = (warp >> 1) & 1;
      const auto tile = [&](auto is_dk) {
        constexpr bool DKO = decltype(is_dk)::value;
        constexpr int KD = DKO ? DV : DK, ND = DKO ? DK : DV;          // contracted with dS; columns
        constexpr int AP = DKO ? VP : KP, BP = DKO ? KP : VP, NT8 = ND / 16;
        const uint32_t ta = DKO ? uv : uk, tb = DKO ? uq : uo, ts = DKO ? ud : up;
        const int n0 = half * (ND / 2), nd = DKO ? p.kd : p.vd;
          float o[2][NT8][4] = {};
#pragma unroll 2
          for (int kk = 0; kk < KD / 16; ++kk) {
            uint32_t a[2][4];
            ldsm(a[0], ta + r0 * AP + ((DKO ? lav : lak) ^ (kk * 32)));
            ldsm(a[1], ta + r1 * AP + ((DKO ? lav : lak) ^ (kk * 32)));
#pragma unroll
            for (int s = NS - 1; s >= 0; --s)
#pragma unroll
              for (int n = 0; n < NT8 / 2; ++n) {
                uint32_t b[4];
                if constexpr (DKO) ldsm(b, us + s * Y::SP + (n0 + 16 * n) * VP + (lbv ^ (kk * 32)));
                else ldsm_t(b, us + s * Y::SP + kk * 16 * VP + (lav ^ (n0 * 2 + 32 * n)));
#pragma unroll
                for (int r = 0; r < 2; ++r) { mma16(o[r][2 * n], a[r], b[0], b[1]); mma16(o[r][2 * n + 1], a[r], b[2], b[3]); }
              }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = (r ? r1 : r0) + gr;
            const float w0 = gs.wt[row].y, w1 = gs.wt[row + 8].y;
#pragma unroll
            for (int n = 0; n < NT8; ++n) { o[r][n][0] *= w0; o[r][n][1] *= w0; o[r][n][2] *= w1; o[r][n][3] *= w1; }
          }
          if constexpr (DKO && GATE) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf) {
                const int row = (r ? r1 : r0) + gr + 8 * hf;
                float x = 0.f;
#pragma unroll
                for (int n = 0; n < NT8; ++n) {
                  uint32_t kk;
                  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(kk) : "r"(at16<KP>(uk, row, n0 / 8 + n) + 4 * tq));
                  const float2 y = pair_of(kk);
                  x = fmaf(o[r][n][2 * hf], y.x, fmaf(o[r][n][2 * hf + 1], y.y, x));
                }
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                if (tq == 0) bd_[(i & 1) * 128 + half * 64 + row] = x;
              }
          }
#pragma unroll 1
          for (int ki = r0; ki < 64 && ki < nv; ki += 16) {
            uint32_t a[2][4];
            ldsm_t(a[0], ts + ki * 128 + (lbp ^ (r0 * 2)));
            const bool both = ki >= r1;
            if (both) ldsm_t(a[1], ts + ki * 128 + (lbp ^ (r1 * 2)));
            uint32_t b[NT8 / 2][4];
            bool odd = false;
#pragma unroll
            for (int n = 0; n < NT8 / 2; ++n) {
              ldsm_t(b[n], tb + ki * BP + ((DKO ? lak : lav) ^ (n0 * 2 + 32 * n)));
              odd = odd || not_finite(b[n]);
            }
            odd = __any_sync(0xffffffffu, odd);
            if (odd && ki == r0) {
              diagonal_by_sums<BP, NT8, true>(o[0], ts, tb, ki, n0, gr, tq);
            } else {
#pragma unroll
              for (int n = 0; n < NT8 / 2; ++n) { mma16(o[0][2 * n], a[0], b[n][0], b[n][1]); mma16(o[0][2 * n + 1], a[0], b[n][2], b[n][3]); }
            }
            if (odd && ki == r1) {
              diagonal_by_sums<BP, NT8, true>(o[1], ts, tb, ki, n0, gr, tq);
            } else if (both) {
#pragma unroll
              for (int n = 0; n < NT8 / 2; ++n) { mma16(o[1][2 * n], a[1], b[n][0], b[n][1]); mma16(o[1][2 * n + 1], a[1], b[n][2], b[n][3]); }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int row = (r ? r1 : r0) + gr + 8 * hf;
              const int64_t at = ((t0 + row) * p.H + h) * nd + n0;
              if (DKO && q.dk_f32) {
#pragma unroll
                for (int n = 0; n < NT8; ++n)
                  if (row < nv && n0 + 8 * n < nd)
                    *reinterpret_cast<float2*>((float*)q.dk + at + 8 * n + 2 * tq) = make_float2(o[r][n][2 * hf], o[r][n][2 * hf + 1]);
              } else {
#pragma unroll
                for (int g = 0; g < NT8; g += 4) {
                  uint32_t v[4];
#pragma unroll
                  for (int n = 0; n < 4; ++n) v[n] = pack_bf16x2(o[r][g + n][2 * hf], o[r][g + n][2 * hf + 1]);
                  transpose4(v, tq);
                  if (row < nv && n0 + 8 * (g + tq) < nd)
                    *reinterpret_cast<uint4*>((bf16*)(DKO ? q.dk : q.dv) + at + 8 * (g + tq)) = make_uint4(v[0], v[1], v[2], v[3]);
                }
              }
            }
      };
      if (warp >> 2) tile(std::true_type()); else tile(std::false_type());
    }
    // dS = exp(lam_L) dS + (exp(lam_i) Q)^T dO
    const float all = gs.wt[63].x;
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[m][n][e] *= all;
#pragma unroll 1
    for (int kk = 0; kk < 64 && kk < nv; kk += 16) {
      const int j = kk + 2 * tq;
      const float w[4] = {gs.wt[j].x, gs.wt[j + 1].x, gs.wt[j + 8].x, gs.wt[j + 9].x};
      uint32_t z[MR][2][4];
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        uint32_t a[4];
        ldsm_t(a, uq + kk * KP + (lbk ^ (ur * 2 + 32 * m)));
        weighted<2>(z[m], a, w);
      }
#pragma unroll
      for (int n = 0; n < NV / 2; ++n) {
        uint32_t b[4];
        ldsm_t(b, uo + kk * VP + (lav ^ (uc * 2 + 32 * n)));
#pragma unroll
        for (int s = 1; s >= 0; --s)
#pragma unroll
          for (int m = 0; m < MR; ++m) { mma16(st[m][2 * n], z[m][s], b[0], b[1]); mma16(st[m][2 * n + 1], z[m][s], b[2], b[3]); }
      }
    }
  }
  if constexpr (GATE) {
    __syncthreads();
    if (warp == 7 && chunks) gates(0);
  }
  if (p.fin && run.first)
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = ur + 16 * m + gr + 8 * (e / 2), c = uc + 8 * n + 2 * tq + e % 2;
          if (c < p.vd && k < p.kd) st_any(p.fin, !p.fin_f32, sh * dd + k * p.ik + c * p.ic, st[m][n][e]);
        }
}

template <int KD, int NC, int NU, int NS, bool OUT>
int launch_fast(cudaStream_t stream, Walk p, const char* name) {
  using Y = FLay<KD, NC, OUT>;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(fast_walk_kernel<KD, NC, NU, NS, OUT>, Y::END));
  p.vt = (p.vd + Y::VT - 1) / Y::VT;
  ProfScope ps(name, stream);
  fast_walk_kernel<KD, NC, NU, NS, OUT><<<dim3((unsigned)p.nslots, (unsigned)(p.H * p.vt)), 128, Y::END, stream>>>(p);
  GLA_CHECK_LAUNCH();
  return GLA_OK;
}
template <int DK, int DV, bool GATE>
int launch_back(cudaStream_t stream, const Back& b) {
  using Y = BLay<DK, DV, GATE ? 2 : 1>;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(fast_back_kernel<DK, DV, GATE>, Y::END));
  ProfScope ps("decay_back_kernel", stream);
  fast_back_kernel<DK, DV, GATE><<<dim3((unsigned)b.w.nslots, (unsigned)b.w.H), 256, Y::END, stream>>>(b);
  GLA_CHECK_LAUNCH();
  return GLA_OK;
}
// planes of the weighted values and of the state: 2, 1 | 3, 1 (a state that leaves in float32) | 2, 2 (with the gates' gradient)
enum FastKind { F_ONE = 0, F_STATE = 1, F_FINE = 2, F_SUMS = 3, F_SUMS_STATE = 4 };
int fast_walk(cudaStream_t, const Walk&, int kind, const char* name);
int fast_back(cudaStream_t, const Back&, bool gate);
unsigned int bad_offsets_fast();

}  // namespace decay
}  // namespace gla
