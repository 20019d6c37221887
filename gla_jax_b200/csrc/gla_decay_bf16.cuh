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
template <int D, int NT>
__device__ __forceinline__ void fetch_tile(uint32_t dst, const void* src, int64_t row0, int64_t step, int nv, int d) {
  constexpr int C8 = D / 8;
#pragma unroll
  for (int j = 0; j < 64 * C8 / NT; ++j) {
    const int i = threadIdx.x + NT * j, r = i / C8, c = i % C8;
    const bool in = r < nv && c * 8 < d;
    cp16(at16<2 * D>(dst, r, c), (const bf16*)src + (in ? row0 + r * step + c * 8 : 0), in);
  }
}
// fragments: A [m][k], A [k][m], B [n][k] and B [k][n], 16 x 16 at (row, column) of a tile
template <int PITCH> __device__ __forceinline__ void frag_a(uint32_t (&a)[4], uint32_t t, int m, int k, int lane) {
  ldsm(a, at16<PITCH>(t, m + (lane & 15), k / 8 + (lane >> 4)));
}
template <int PITCH> __device__ __forceinline__ void frag_at(uint32_t (&a)[4], uint32_t t, int k, int m, int lane) {
  ldsm_t(a, at16<PITCH>(t, k + (lane & 7) + ((lane >> 4) & 1) * 8, m / 8 + ((lane >> 3) & 1)));
}
template <int PITCH> __device__ __forceinline__ void frag_b(uint32_t (&b)[4], uint32_t t, int n, int k, int lane) {
  ldsm(b, at16<PITCH>(t, n + (lane & 7) + ((lane >> 4) & 1) * 8, k / 8 + ((lane >> 3) & 1)));
}
template <int PITCH> __device__ __forceinline__ void frag_bt(uint32_t (&b)[4], uint32_t t, int k, int n, int lane) {
  ldsm_t(b, at16<PITCH>(t, k + (lane & 15), n / 8 + (lane >> 4)));
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

// The gates of a chunk of 64 by one warp: two rows a lane.  lam: running sums, base 2, as two floats; wt: exp(lam_i) and
// exp(lam_L - lam_i).  Returns the chunk's sum (base 2).
__device__ __forceinline__ float2 gates_of(const Walk& p, int64_t t0, int nv, int h, int lane) {
  float2 g = make_float2(0.f, 0.f);
  if (2 * lane < nv) g.x = p.g[(t0 + 2 * lane) * p.gt + h];
  if (2 * lane + 1 < nv) g.y = p.g[(t0 + 2 * lane + 1) * p.gt + h];
  return g;
}
__device__ __forceinline__ double scan_gates(float2 g, float2* lam, float2* wt, int lane) {
  // exp of less than -200 is 0 either way; -inf would leave inf - inf
  const double a = (double)(g.x < -200.f ? -200.f : g.x) * 1.4426950408889634, b = (double)(g.y < -200.f ? -200.f : g.y) * 1.4426950408889634;
  double inc = a + b;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  const double all = __shfl_sync(0xffffffffu, inc, 31);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double v = i ? inc : inc - b;
    const float hi = (float)v;
    lam[2 * lane + i] = make_float2(hi, (float)(v - hi));
    wt[2 * lane + i] = make_float2(exp2f((float)v), exp2f((float)(all - v)));
  }
  return all;
}
__device__ __forceinline__ float decay_of(float2 i, float2 j) { return exp2f((i.x - j.x) + (i.y - j.y)); }

template <int KD, int NC, bool OUT>
struct FLay {
  static constexpr int VT = 64 * NC, NT = 128;
  static constexpr int PK = 128 * KD, PV = 128 * VT, STAGE = (OUT ? 2 : 1) * PK + PV;
  static constexpr int P0 = 2 * STAGE, LAM = P0 + (OUT ? 8192 : 0), WT = LAM + 1024, RD = WT + 1024, END = RD + (OUT ? 1024 : 0);
};

// KD: features; NC: groups of 16 value columns of a warp; NU: planes of the weighted values (3: and exact additions); NS:
// planes of the state as an operand
template <int KD, int NC, int NU, int NS, bool OUT>
__global__ void __launch_bounds__(128, 2) fast_walk_kernel(const Walk p) {
  using Y = FLay<KD, NC, OUT>;
  constexpr int KT = KD / 8, QP = 2 * KD, VP = 2 * Y::VT;
  extern __shared__ __align__(128) uint8_t sm[];
  float2* lam_ = reinterpret_cast<float2*>(sm + Y::LAM);
  float2* wt_ = reinterpret_cast<float2*>(sm + Y::WT);
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

  const int Hq = p.H / p.gq, Hk = p.H / p.gk, Hv = p.H / p.gv, Hr = p.r ? p.H / p.gr : 1;
  const int len = (int)(run.hi - run.lo), chunks = (len + 63) / 64;
  const uint32_t base = sm32(sm);
  // chunk i of the walk; backwards in time (sums only) from the last one
  const auto first_of = [&](int i) { return 64 * (p.rev ? chunks - 1 - i : i); };
  const auto fetch = [&](int i) {
    const int c0 = first_of(i), nv = len - c0 < 64 ? len - c0 : 64;
    const int64_t t0 = run.base + run.lo + c0;
    const uint32_t s = base + (i & 1) * Y::STAGE;
    fetch_tile<KD, 128>(s, p.k, (t0 * Hk + h / p.gk) * p.kd, (int64_t)Hk * p.kd, nv, p.kd);
    fetch_tile<Y::VT, 128>(s + Y::PK, p.v, (t0 * Hv + h / p.gv) * p.vd + cbase, (int64_t)Hv * p.vd, nv, p.vd - cbase);
    if constexpr (OUT) fetch_tile<KD, 128>(s + Y::PK + Y::PV, p.q, (t0 * Hq + h / p.gq) * p.kd, (int64_t)Hq * p.kd, nv, p.kd);
  };
  double total = 0.0;
  if (chunks) {
    fetch(0);
    if (warp == 0) {
      const int c0 = first_of(0);
      total += scan_gates(gates_of(p, run.base + run.lo + c0, len - c0 < 64 ? len - c0 : 64, h, lane), lam_, wt_, lane);
    }
  }
  cp_commit();
  for (int i = 0; i < chunks; ++i) {
    const int c0 = first_of(i), nv = len - c0 < 64 ? len - c0 : 64;
    const int64_t t0 = run.base + run.lo + c0;
    const uint32_t uk = base + (i & 1) * Y::STAGE, uv = uk + Y::PK, uq = uv + Y::PV, up = base + Y::P0;
    const float2 *lam = lam_ + 64 * (i & 1), *wt = wt_ + 64 * (i & 1);
    cp_wait<0>();
    __syncthreads();                 // this chunk is here, and nobody reads the other stage any more
    float2 gn = make_float2(0.f, 0.f);
    if (i + 1 < chunks) {
      fetch(i + 1);
      if (warp == 0) {
        const int n0 = first_of(i + 1);
        gn = gates_of(p, run.base + run.lo + n0, len - n0 < 64 ? len - n0 : 64, h, lane);
      }
    }
    cp_commit();
    if constexpr (OUT) {
      if (p.r && i > 0 && tid < 64) {
        // the row sums of the chunk before (a whole one)
        p.rdot[(vt * (p.cu ? p.T : p.nseq * p.T) + t0 - 64 + tid) * p.H + h] = (rd[tid] + rd[64 + tid]) + (rd[128 + tid] + rd[192 + tid]);
      }
      // scores in blocks of 16 x 16: rows 48.. by two warps, 32.. by one, 16.. and 0.. by one
      const auto scores = [&](auto nb, int mi, int nj) {
        constexpr int NB = decltype(nb)::value;
        float c[NB][2][4] = {};
#pragma unroll
        for (int kk = 0; kk < KD / 16; ++kk) {
          uint32_t a[4];
          frag_a<QP>(a, uq, mi * 16, kk * 16, lane);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            uint32_t x[4];
            frag_b<QP>(x, uk, (nj + b) * 16, kk * 16, lane);
            mma16(c[b][0], a, x[0], x[1]);
            mma16(c[b][1], a, x[2], x[3]);
          }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const int r = mi * 16 + gr + 4 * e, j = (nj + b) * 16 + n * 8 + 2 * tq;
              const float2 lr = lam[r];
              const float x = j <= r ? c[b][n][e] * decay_of(lr, lam[j]) : 0.f, y = j + 1 <= r ? c[b][n][e + 1] * decay_of(lr, lam[j + 1]) : 0.f;
              const uint32_t z = pack_bf16x2(x, y);
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(at16<128>(up, r, j / 8) + (j % 8) * 2), "r"(z) : "memory");
            }
      };
      if (warp == 0) scores(std::integral_constant<int, 2>(), 3, 0);
      else if (warp == 1) scores(std::integral_constant<int, 2>(), 3, 2);
      else if (warp == 2) scores(std::integral_constant<int, 3>(), 2, 0);
      else { scores(std::integral_constant<int, 2>(), 1, 0); scores(std::integral_constant<int, 1>(), 0, 0); }
    }
    if (warp == 0 && i + 1 < chunks) total += scan_gates(gn, lam_ + 64 * ((i + 1) & 1), wt_ + 64 * ((i + 1) & 1), lane);
    if constexpr (OUT) {
      __syncthreads();
#pragma unroll 1
      for (int m = 0; m < 64 && m < nv; m += 32) {
        float o[2][2 * NC][4];
        const auto inter = [&](float (&x)[2][2 * NC][4]) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < 2 * NC; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[r][n][e] = 0.f;
#pragma unroll
          for (int kk = 0; kk < KD / 16; ++kk) {
            uint32_t a[2][4];
            frag_a<QP>(a[0], uq, m, kk * 16, lane);
            frag_a<QP>(a[1], uq, m + 16, kk * 16, lane);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
              uint32_t b0[NS], b1[NS], b2[NS], b3[NS];
              planes<NS>(st[n][2 * kk][0], st[n][2 * kk][1], b0);
              planes<NS>(st[n][2 * kk + 1][0], st[n][2 * kk + 1][1], b1);
              planes<NS>(st[n][2 * kk][2], st[n][2 * kk][3], b2);
              planes<NS>(st[n][2 * kk + 1][2], st[n][2 * kk + 1][3], b3);
#pragma unroll
              for (int s = NS - 1; s >= 0; --s)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  mma16(x[r][2 * n], a[r], b0[s], b1[s]);
                  mma16(x[r][2 * n + 1], a[r], b2[s], b3[s]);
                }
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float w0 = wt[m + 16 * r + gr].x, w1 = wt[m + 16 * r + gr + 8].x;
#pragma unroll
            for (int n = 0; n < 2 * NC; ++n) { x[r][n][0] *= w0; x[r][n][1] *= w0; x[r][n][2] *= w1; x[r][n][3] *= w1; }
          }
        };
        inter(o);
        if (p.r) {
          // the rows' products with what comes from before the chunk
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float dot[2] = {0.f, 0.f};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int row = m + 16 * r + gr + 8 * half;
              if (row < nv) {
                const int64_t ra = ((t0 + row) * Hr + h / p.gr) * p.vd + cw + 2 * tq;
#pragma unroll
                for (int n = 0; n < 2 * NC; ++n)
                  if (cw + 8 * n < p.vd) {
                    const float2 x = pair_of(__ldg((const unsigned int*)((const bf16*)p.r + ra + 8 * n)));
                    dot[half] = fmaf(o[r][n][2 * half], x.x, fmaf(o[r][n][2 * half + 1], x.y, dot[half]));
                  }
              }
              dot[half] += __shfl_xor_sync(0xffffffffu, dot[half], 1);
              dot[half] += __shfl_xor_sync(0xffffffffu, dot[half], 2);
              if (tq == 0) rd[warp * 64 + row] = dot[half];
            }
          }
        }
        for (int kj = 0; kj <= m / 16 + 1; ++kj) {
          uint32_t a[2][4], b[NC][4];
#pragma unroll
          for (int n = 0; n < NC; ++n) frag_bt<VP>(b[n], uv, kj * 16, cl + 16 * n, lane);
          frag_a<128>(a[1], up, m + 16, kj * 16, lane);
#pragma unroll
          for (int n = 0; n < NC; ++n) { mma16(o[1][2 * n], a[1], b[n][0], b[n][1]); mma16(o[1][2 * n + 1], a[1], b[n][2], b[n][3]); }
          if (kj <= m / 16) {
            frag_a<128>(a[0], up, m, kj * 16, lane);
#pragma unroll
            for (int n = 0; n < NC; ++n) { mma16(o[0][2 * n], a[0], b[n][0], b[n][1]); mma16(o[0][2 * n + 1], a[0], b[n][2], b[n][3]); }
          }
        }
        // A value that is not finite meets the zeros above the diagonal (0 x inf); the recurrence has it at its own token
        // and after only, so what is not finite is summed again over j <= i
        float bad = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < 2 * NC; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad = fmaf(o[r][n][e], 0.f, bad);
        if (__any_sync(0xffffffffu, bad != 0.f)) {
          float keep[2][2 * NC][4];
          inter(keep);
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < 2 * NC; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(fabsf(o[r][n][e]) <= 3.402823466e38f)) {
                  const int row = m + 16 * r + gr + 8 * (e / 2), c = cl + 8 * n + 2 * tq + e % 2;
                  float x = keep[r][n][e];
#pragma unroll 1
                  for (int j = 0; j <= row; ++j) {
                    uint16_t s, v;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s) : "r"(at16<128>(up, row, j / 8) + (j % 8) * 2));
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at16<VP>(uv, j, c / 8) + (c % 8) * 2));
                    x = fmaf(__uint_as_float((uint32_t)s << 16), __uint_as_float((uint32_t)v << 16), x);
                  }
                  o[r][n][e] = x;
                }
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int row = m + 16 * r + gr + 8 * half;
            if (row < nv) {
              const int64_t at = ((t0 + row) * p.H + h) * p.vd + cw + 2 * tq;
#pragma unroll
              for (int n = 0; n < 2 * NC; ++n)
                if (cw + 8 * n < p.vd) {
                  const float x = o[r][n][2 * half], y = o[r][n][2 * half + 1];
                  if (p.out_f32) *reinterpret_cast<float2*>((float*)p.out + at + 8 * n) = make_float2(x, y);
                  else *reinterpret_cast<uint32_t*>((bf16*)p.out + at + 8 * n) = pack_bf16x2(x, y);
                }
            }
          }
      }
    } else {
      // (the gates of the next chunk are read behind the next barrier)
    }
    // the state: st = exp(lam_L) st + (w V)^T K, backwards in time with exp(lam_i) as weights
    const float all = wt[63].x;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[n][j][e] *= all;
#pragma unroll 1
    for (int kk = 0; kk < 64 && kk < nv; kk += 16) {
      const int j = kk + 2 * tq;
      const float w[4] = {p.rev ? wt[j].x : wt[j].y, p.rev ? wt[j + 1].x : wt[j + 1].y, p.rev ? wt[j + 8].x : wt[j + 8].y,
                          p.rev ? wt[j + 9].x : wt[j + 9].y};
      uint32_t z[NC][NU][4];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        uint32_t a[4];
        frag_at<VP>(a, uv, kk, cl + 16 * n, lane);
        weighted<NU>(z[n], a, w);
      }
#pragma unroll
      for (int t = 0; t < KD / 16; ++t) {
        uint32_t b[1][4];
        frag_bt<QP>(b[0], uk, kk, t * 16, lane);
#pragma unroll
        for (int n = 0; n < NC; ++n) mma_planes<NU, 1, (NU > 2)>(st[n][2 * t], st[n][2 * t + 1], z[n], b);
      }
    }
  }

  if constexpr (OUT) {
    if (p.r && chunks) {
      __syncthreads();
      const int c0 = 64 * (chunks - 1);
      if (tid < len - c0)
        p.rdot[(vt * (p.cu ? p.T : p.nseq * p.T) + run.base + run.lo + c0 + tid) * p.H + h] = (rd[tid] + rd[64 + tid]) + (rd[128 + tid] + rd[192 + tid]);
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
  static constexpr int S0 = 2 * STAGE, SP = DK * DV * 2, P0 = S0 + NS * SP, D0 = P0 + 8192, LAM = D0 + 8192, WT = LAM + 1024;
  static constexpr int RS = WT + 1024, CS = RS + 2 * 2048, BD = CS + 2 * 1024, RED = BD + 2 * 512, END = RED + 64;
};
template <int DK, int DV, bool GATE>
__global__ void __launch_bounds__(256, 1) fast_back_kernel(const Back q) {
  constexpr int NS = GATE ? 2 : 1;
  using Y = BLay<DK, DV, NS>;
  constexpr int KP = 2 * DK, VP = 2 * DV, MR = DK / 64, NV = DV / 16;   // update: MR x 16 rows and NV tiles of 8 columns per warp
  const Walk& p = q.w;
  extern __shared__ __align__(128) uint8_t sm[];
  float2* lam_ = reinterpret_cast<float2*>(sm + Y::LAM);
  float2* wt_ = reinterpret_cast<float2*>(sm + Y::WT);
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
  const auto fetch = [&](int i) {
    const int nv = len - 64 * i < 64 ? len - 64 * i : 64;
    const int64_t t0 = run.base + run.lo + 64 * i;
    const uint32_t s = base + (i & 1) * Y::STAGE;
    const int64_t rk = (t0 * Hq + h / p.gq) * p.kd, rv = (t0 * p.H + h) * p.vd;
    fetch_tile<DK, 256>(s, p.q, rk, (int64_t)Hq * p.kd, nv, p.kd);
    fetch_tile<DK, 256>(s + Y::TK, p.k, rk, (int64_t)Hq * p.kd, nv, p.kd);
    fetch_tile<DV, 256>(s + 2 * Y::TK, p.v, rv, (int64_t)p.H * p.vd, nv, p.vd);
    fetch_tile<DV, 256>(s + 2 * Y::TK + Y::TV, q.dout, rv, (int64_t)p.H * p.vd, nv, p.vd);
  };
  if (chunks) {
    fetch(chunks - 1);
    if (warp == 0)
      scan_gates(gates_of(p, run.base + run.lo + 64 * (chunks - 1), len - 64 * (chunks - 1), h, lane), lam_ + 64 * ((chunks - 1) & 1),
                 wt_ + 64 * ((chunks - 1) & 1), lane);
  }
  cp_commit();
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
    const float2 *lam = lam_ + 64 * (i & 1), *wt = wt_ + 64 * (i & 1);
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
      const int mi = u < 2 ? 0 : u < 6 ? 1 : u < 12 ? 2 : 3, nt = u - mi * (mi + 1);
      float c[4] = {}, d[4] = {};
#pragma unroll
      for (int kk = 0; kk < DK / 32; ++kk) {
        uint32_t a[4], a2[4], b[4];
        ldsm(b, at16<KP>(uk, nt * 8 + (lane & 7), kk * 4 + (lane >> 3)));
        frag_a<KP>(a, uq, mi * 16, kk * 32, lane);
        frag_a<KP>(a2, uq, mi * 16, kk * 32 + 16, lane);
        mma16(c, a, b[0], b[1]);
        mma16(c, a2, b[2], b[3]);
      }
#pragma unroll
      for (int kk = 0; kk < DV / 32; ++kk) {
        uint32_t a[4], a2[4], b[4];
        ldsm(b, at16<VP>(uv, nt * 8 + (lane & 7), kk * 4 + (lane >> 3)));
        frag_a<VP>(a, uo, mi * 16, kk * 32, lane);
        frag_a<VP>(a2, uo, mi * 16, kk * 32 + 16, lane);
        mma16(d, a, b[0], b[1]);
        mma16(d, a2, b[2], b[3]);
      }
      float cm[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int r = mi * 16 + gr + 4 * e, j = nt * 8 + 2 * tq;
        const float w0 = j <= r ? decay_of(lam[r], lam[j]) : 0.f, w1 = j + 1 <= r ? decay_of(lam[r], lam[j + 1]) : 0.f;
        const float x0 = j <= r ? c[e] * w0 : 0.f, x1 = j + 1 <= r ? c[e + 1] * w1 : 0.f;
        const uint32_t at = at16<128>(0, r, nt) + 4 * tq;
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(up + at), "r"(pack_bf16x2(x0, x1)) : "memory");
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(ud + at), "r"(pack_bf16x2(j <= r ? d[e] * w0 : 0.f, j + 1 <= r ? d[e + 1] * w1 : 0.f)) : "memory");
        if constexpr (GATE) {
          const float m0 = j <= r ? x0 * d[e] : 0.f, m1 = j + 1 <= r ? x1 * d[e + 1] : 0.f;
          cm[0] += m0;
          cm[1] += m1;
          float x = m0 + m1;
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (tq == 0) rs_[(i & 1) * 512 + nt * 64 + r] = x;
        }
      }
      if constexpr (GATE) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) { cm[0] += __shfl_xor_sync(0xffffffffu, cm[0], s); cm[1] += __shfl_xor_sync(0xffffffffu, cm[1], s); }
        if (gr == 0) *reinterpret_cast<float2*>(cs_ + (i & 1) * 256 + mi * 64 + nt * 8 + 2 * tq) = make_float2(cm[0], cm[1]);
      }
    }
    if (warp == 7) {
      if (i > 0) scan_gates(gn, lam_ + 64 * ((i - 1) & 1), wt_ + 64 * ((i - 1) & 1), lane);
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
        float o[2][NT8][4];
        const auto inter = [&](float (&x)[2][NT8][4]) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < NT8; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) x[r][n][e] = 0.f;
#pragma unroll 2
          for (int kk = 0; kk < KD / 16; ++kk) {
            uint32_t a[2][4];
            frag_a<AP>(a[0], ta, r0, kk * 16, lane);
            frag_a<AP>(a[1], ta, r1, kk * 16, lane);
#pragma unroll
            for (int n = 0; n < NT8 / 2; ++n)
#pragma unroll
              for (int s = NS - 1; s >= 0; --s) {
                uint32_t b[4];
                if constexpr (DKO) frag_b<VP>(b, us + s * Y::SP, n0 + 16 * n, kk * 16, lane);
                else frag_bt<VP>(b, us + s * Y::SP, kk * 16, n0 + 16 * n, lane);
#pragma unroll
                for (int r = 0; r < 2; ++r) { mma16(x[r][2 * n], a[r], b[0], b[1]); mma16(x[r][2 * n + 1], a[r], b[2], b[3]); }
              }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = (r ? r1 : r0) + gr;
            const float w0 = wt[row].y, w1 = wt[row + 8].y;
#pragma unroll
            for (int n = 0; n < NT8; ++n) { x[r][n][0] *= w0; x[r][n][1] *= w0; x[r][n][2] *= w1; x[r][n][3] *= w1; }
          }
        };
        inter(o);
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
        for (int ki = r0 / 16; ki < 4 && ki * 16 < nv; ++ki) {
          uint32_t a[2][4];
          frag_at<128>(a[0], ts, ki * 16, r0, lane);
          if (ki * 16 >= r1) frag_at<128>(a[1], ts, ki * 16, r1, lane);
#pragma unroll
          for (int n = 0; n < NT8 / 2; ++n) {
            uint32_t b[4];
            frag_bt<BP>(b, tb, ki * 16, n0 + 16 * n, lane);
            mma16(o[0][2 * n], a[0], b[0], b[1]);
            mma16(o[0][2 * n + 1], a[0], b[2], b[3]);
            if (ki * 16 >= r1) { mma16(o[1][2 * n], a[1], b[0], b[1]); mma16(o[1][2 * n + 1], a[1], b[2], b[3]); }
          }
        }
        float bad = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NT8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) bad = fmaf(o[r][n][e], 0.f, bad);
        if (__any_sync(0xffffffffu, bad != 0.f)) {
          // as in the forward: what is not finite is summed again, here over i >= j
          float keep[2][NT8][4];
          inter(keep);
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < NT8; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (!(fabsf(o[r][n][e]) <= 3.402823466e38f)) {
                  const int j = (r ? r1 : r0) + gr + 8 * (e / 2), c = n0 + 8 * n + 2 * tq + e % 2;
                  float x = keep[r][n][e];
#pragma unroll 1
                  for (int t = j; t < nv; ++t) {
                    uint16_t s, v;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(s) : "r"(at16<128>(ts, t, j / 8) + (j % 8) * 2));
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at16<BP>(tb, t, c / 8) + (c % 8) * 2));
                    x = fmaf(__uint_as_float((uint32_t)s << 16), __uint_as_float((uint32_t)v << 16), x);
                  }
                  o[r][n][e] = x;
                }
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const int row = (r ? r1 : r0) + gr + 8 * hf;
            if (row < nv) {
              const int64_t at = ((t0 + row) * p.H + h) * nd + n0 + 2 * tq;
#pragma unroll
              for (int n = 0; n < NT8; ++n)
                if (n0 + 8 * n < nd) {
                  const float x = o[r][n][2 * hf], y = o[r][n][2 * hf + 1];
                  if (DKO && q.dk_f32) *reinterpret_cast<float2*>((float*)q.dk + at + 8 * n) = make_float2(x, y);
                  else *reinterpret_cast<uint32_t*>((bf16*)(DKO ? q.dk : q.dv) + at + 8 * n) = pack_bf16x2(x, y);
                }
            }
          }
      };
      if (warp >> 2) tile(std::true_type()); else tile(std::false_type());
    }
    // dS = exp(lam_L) dS + (exp(lam_i) Q)^T dO
    const float all = wt[63].x;
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[m][n][e] *= all;
#pragma unroll 1
    for (int kk = 0; kk < 64 && kk < nv; kk += 16) {
      const int j = kk + 2 * tq;
      const float w[4] = {wt[j].x, wt[j + 1].x, wt[j + 8].x, wt[j + 9].x};
      uint32_t z[MR][2][4];
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        uint32_t a[4];
        frag_at<KP>(a, uq, kk, ur + 16 * m, lane);
        weighted<2>(z[m], a, w);
      }
#pragma unroll
      for (int n = 0; n < NV / 2; ++n) {
        uint32_t b[1][4];
        frag_bt<VP>(b[0], uo, kk, uc + 16 * n, lane);
#pragma unroll
        for (int m = 0; m < MR; ++m) mma_planes<2, 1, false>(st[m][2 * n], st[m][2 * n + 1], z[m], b);
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
