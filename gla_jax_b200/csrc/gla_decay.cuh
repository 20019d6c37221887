// Linear attention with one decay per head: S_t = exp(g_t) S_{t-1} + k_t (x) v_t, o_t = q_t S_t, g a number per token and
// value head (gla_chunk_fwd has one per key feature).
//
// One kernel walks a run of tokens, L at a time, with the state in registers.  lam = running sum of g inside the chunk:
//   O  = tril(Q K^T . exp(lam_i - lam_j)) V + exp(lam_i) (Q S)          S <- exp(lam_L) S + V^T (exp(lam_L - lam_j) K)
// The decay is a scalar, so it multiplies scores and never an operand that a tensor map could have fetched: no anchor and
// no range of the weights to guard, every exp(lam_i - lam_j) is formed as it stands (lam in 64 bits, kept as two floats, so
// that a gate which resets the state costs the later weights nothing).
//
// Why register operands.  A warp owns 16 value columns of the state, transposed (16 x KD accumulators of V^T K).  Two
// neighbouring accumulators of a row are what a lane has to hold of B in Q S, so the state goes from one product into the
// other without shared memory, and nothing but the scores is exchanged between warps.
//
// The same kernel is the backward: with roles exchanged,
//   dq = walk(q: dO, k: v, v: k, state: S^T)           forwards
//   dv = walk(q: k, k: q, v: dO, state: dS)            backwards in time, the gate of the next token at each step
//   dk = walk(q: v, k: dO, v: q, state: dS^T)          backwards
// and dg_t = sum over i >= t > j of w_ij (q_i k_j)(do_i v_j), pairs of a chunk one by one, the others by what comes from outside it:
//   dg_t = <S_T, dS_T> + sum over i >= t of (a_i - b_i) + the chunk's pairs,   a = q . (dq from before), b = k . (dk from behind)
//
// Types.  bf16 operands go to the tensor cores as they are, float32 ones as three bf16 planes (8 + 8 + 8 bits).  What the
// kernel forms itself (scores, the state as an operand, weighted values) is split into as many planes as the mode says.
#pragma once
#include "gla_common.cuh"
#include "tc_ptx.cuh"
#include "tma_maps.cuh"

namespace gla {
namespace decay {

using tc::pack_bf16x2;

// one: bf16 in and out, scores and the state as an operand rounded once to 8 bits (2^-9 of each term of sums over 64 and more), the
//   state summed from values in two planes: what it holds is there for all later tokens (with one plane 2.3e-3 of its norm off as it
//   leaves, with two its own rounding, 1.7e-3; 4 x 4096 tokens, 4 heads of 256 x 256: 327 -> 354 us)
// state: the same with the state updated from three planes, for a state that leaves in float32
// fine: formed operands in two planes (2^-17), for gradients whose row sums cancel in dg
// full: float32 in and out
enum ModeId { M_ONE = 0, M_STATE = 1, M_FINE = 2, M_FULL = 3 };
template <int M> struct Mode {
  static constexpr int NI = M == M_FULL ? 3 : 1;                         // planes of q, k, v
  static constexpr int NF = M == M_FULL ? 3 : M == M_FINE ? 2 : 1;       // of scores and of the state as an operand
  static constexpr int NU = M == M_FULL || M == M_STATE ? 3 : 2;         // of weighted values
  static constexpr int L = M == M_FULL ? 32 : 64;
  static constexpr bool EXO = M >= M_FINE, EXU = M >= M_STATE;           // 16 of K summed from zero, then added in float32
};

struct Walk {
  const void *q, *k, *v;            // [token][heads][kd], [token][heads][kd], [token][heads][vd]
  int gq, gk, gv;                   // value heads per head of each
  int H, kd, vd, vt;                // value heads, actual sizes, tiles of value columns
  const float* g;                   // [token][H] (gt = H), or [H] (gt = 0)
  int64_t gt;
  const int* cu;                    // packed offsets (rising from 0 to at most T), or NULL: sequence s holds tokens [s T, (s + 1) T)
  int64_t T, nseq, seg, nslots;     // tokens of a sequence (of all, packed), sequences, tokens of a run, runs
  int rev;
  const void* init;                 // entering state, element (k, c) of [s][h] at k ik + c ic
  void* fin;                        // leaving state, the same strides; may be NULL
  float* fin32;                     // the same in float32; may be NULL
  int64_t ik, ic;
  int init_f32, fin_f32;
  float* seg_state;                 // [slot][H][vd][kd]: what a run adds (first pass), then the state that enters it
  int64_t sk, sc;                   // strides in it that the walks of gla_decay_tc.cuh read the entering state with
  double* seg_total;                // [slot][H]: log2 of a run's decay
  void* out;                        // [token][H][vd]
  int out_f32;
  const void* r;                    // rows multiplied into rdot with what comes from outside the chunk: [token][heads][vd]; may be NULL
  int gr;
  float* rdot;                      // [vt][token][H]
};

// Which run a block has.  Packed: the axis is cut at multiples of `seg`, slot s + (start of the run / seg), so that the slot
// number alone tells sequence and run without a table (at most nseq + ceil(T / seg) slots, some of them empty).
struct Run {
  int64_t s, base, lo, hi, a, b;    // sequence; tokens [base + lo, base + hi) of the sequence's [base + a, base + b)
  bool any, first, last;            // whether there is one; whether the sequence starts / ends with it
  int64_t zlo, zhi;                 // rows behind the last sequence, to be zeroed
};
__device__ __forceinline__ Run find_run(const Walk& p, int64_t slot) {
  Run r{};
  if (!p.cu) {
    const int64_t per = (p.T + p.seg - 1) / p.seg, i = slot % per;
    r.s = slot / per;
    r.base = r.s * p.T;
    r.a = 0; r.b = p.T;
    r.lo = i * p.seg;
    r.hi = r.lo + p.seg < p.T ? r.lo + p.seg : p.T;
    r.any = true; r.first = i == 0; r.last = r.hi == p.T;
    return r;
  }
  int64_t l = 0, u = p.nseq - 1;                 // the last s with s + cu[s] / seg <= slot
  while (l < u) {
    const int64_t m = (l + u + 1) / 2;
    if (m + p.cu[m] / p.seg <= slot) l = m; else u = m - 1;
  }
  r.s = l;
  r.a = p.cu[l];
  r.b = p.cu[l + 1];
  const int64_t cell = slot - l;
  r.lo = cell * p.seg > r.a ? cell * p.seg : r.a;
  r.hi = (cell + 1) * p.seg < r.b ? (cell + 1) * p.seg : r.b;
  r.first = cell == r.a / p.seg;
  r.any = r.first || r.lo < r.hi;
  if (r.hi < r.lo) r.hi = r.lo;
  r.last = r.any && r.hi == r.b;
  if (l == p.nseq - 1) {
    r.zlo = cell * p.seg > r.b ? cell * p.seg : r.b;
    r.zhi = (cell + 1) * p.seg < p.T ? (cell + 1) * p.seg : p.T;
  }
  return r;
}
__device__ __forceinline__ int64_t slot_of(const Walk& p, int64_t s, int64_t i, int64_t& n) {   // run i of sequence s, of n
  if (!p.cu) {
    n = (p.T + p.seg - 1) / p.seg;
    return s * n + i;
  }
  const int64_t a = p.cu[s], b = p.cu[s + 1], c = a / p.seg;
  n = b > a ? (b - 1) / p.seg - c + 1 : 1;
  return s + c + i;
}

__device__ __forceinline__ uint32_t sm32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// two values into N planes of 8 bits each
template <int N> __device__ __forceinline__ void planes(float x, float y, uint32_t (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = pack_bf16x2(x, y);
    if (i + 1 < N) {
      x -= __uint_as_float(s[i] << 16);
      y -= __uint_as_float(s[i] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ float2 pair_of(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
// c0 and c1 (two tiles of 8 columns) += A B over 16 of K; b[s]: {tile 0: k 0-7, k 8-15, tile 1: k 0-7, k 8-15}.  Products of
// planes below 2^-24 are left out, small ones come first.
template <int NA, int NB, bool EX>
__device__ __forceinline__ void mma_planes(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[NA][4], const uint32_t (&b)[NB][4]) {
  if constexpr (!EX) {
#pragma unroll
    for (int t = NA + NB - 2; t >= 0; --t)
#pragma unroll
      for (int i = 0; i < NA; ++i)
        if (t - i >= 0 && t - i < NB && t <= 2) {
          mma16(c0, a[i], b[t - i][0], b[t - i][1]);
          mma16(c1, a[i], b[t - i][2], b[t - i][3]);
        }
  } else {
    float y0[4] = {}, y1[4] = {};
    mma_planes<NA, NB, false>(y0, y1, a, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) { c0[e] += y0[e]; c1[e] += y1[e]; }
  }
}

template <int MODE, int KD, int NW, bool OUT>
struct Lay {
  using M = Mode<MODE>;
  static constexpr int L = M::L, VT = NW * 16, NT = NW * 32;
  static constexpr int LDK = 2 * KD + 16, LDV = 2 * VT + 16, LDP = 2 * L + 16;    // row pitches in bytes
  static constexpr int PK = L * LDK, PV = L * LDV, PP = L * LDP;                  // planes
  static constexpr int K0 = 0, V0 = K0 + M::NI * PK, Q0 = V0 + M::NI * PV;
  static constexpr int P0 = Q0 + (OUT ? M::NI * PK : 0), LAM = P0 + (OUT ? M::NF * PP : 0);
  static constexpr int WT = LAM + L * 8, RD = WT + L * 8, END = RD + (OUT ? NW * L * 4 : 0);
};

template <int MODE, int D, int LD, int PLANE, int NT>
__device__ __forceinline__ void load_tile(uint8_t* dst, const void* src, int64_t row0, int64_t step, int nv, int d) {
  constexpr int L = Mode<MODE>::L, C8 = D / 8;
  for (int i = threadIdx.x; i < L * C8; i += NT) {
    const int r = i / C8, c = i % C8 * 8;
    const bool in = r < nv && c < d;
    const int64_t e = in ? row0 + r * step + c : 0;
    uint8_t* at = dst + r * LD + c * 2;
    if constexpr (MODE != M_FULL) {
      cp16(sm32(at), (const bf16*)src + e, in);
    } else {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (in) { x = __ldg((const float4*)((const float*)src + e)); y = __ldg((const float4*)((const float*)src + e) + 1); }
      uint32_t s[4][3];
      planes<3>(x.x, x.y, s[0]); planes<3>(x.z, x.w, s[1]); planes<3>(y.x, y.y, s[2]); planes<3>(y.z, y.w, s[3]);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(at + k * PLANE) = make_uint4(s[0][k], s[1][k], s[2][k], s[3][k]);
    }
  }
}
template <int N> __device__ __forceinline__ float sum_planes(const uint8_t* at, int plane) {
  float x = 0.f;
#pragma unroll
  for (int i = N - 1; i >= 0; --i) x += __bfloat162float(*reinterpret_cast<const bf16*>(at + i * plane));
  return x;
}

// Up to three walks side by side (blockIdx.z): those of a backward do not wait for one another.
struct Walks { Walk w[3]; };
template <int MODE, int KD, int NW, bool OUT>
__global__ void __launch_bounds__(NW * 32, KD <= 128 && MODE <= M_STATE ? 16 / NW : 1) walk_kernel(const __grid_constant__ Walks all) {
  const Walk& p = all.w[blockIdx.z];
  using M = Mode<MODE>;
  using Y = Lay<MODE, KD, NW, OUT>;
  constexpr int L = Y::L, NT = Y::NT, KT = KD / 8;
  constexpr bool DOTS = MODE >= M_FINE;                        // only a backward's walks make them
  extern __shared__ __align__(16) uint8_t sm[];
  float2* lam = reinterpret_cast<float2*>(sm + Y::LAM);        // running sums, base 2, as two floats
  float2* wt = reinterpret_cast<float2*>(sm + Y::WT);          // exp(lam_i), exp(lam_L - lam_i)
  float* rd = reinterpret_cast<float*>(sm + Y::RD);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, gr = lane / 4, tq = lane % 4;
  const int h = blockIdx.y % p.H, vt = blockIdx.y / p.H;
  const int cbase = vt * Y::VT, cw = cbase + warp * 16;        // first value column of the block, of the warp
  grid_dep_launch();
  const Run run = find_run(p, blockIdx.x);
  if constexpr (OUT) {
    if (run.zlo < run.zhi) {
      const int w = p.vd - cbase < Y::VT ? p.vd - cbase : Y::VT;
      for (int64_t i = tid; i < (run.zhi - run.zlo) * w; i += NT)
        st_any(p.out, !p.out_f32, ((run.zlo + i / w) * p.H + h) * p.vd + cbase + i % w, 0.f);
    }
  }
  if (!run.any) return;
  // the run that the sequence is left through has nobody to pass its sum to
  if (!OUT && (p.rev ? run.first : run.last)) return;

  const int64_t sh = run.s * p.H + h, dd = (int64_t)p.kd * p.vd, slot_h = (int64_t)blockIdx.x * p.H + h;
  float st[KT][4];
#pragma unroll
  for (int j = 0; j < KT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = cw + gr + 8 * (e / 2), k = 8 * j + 2 * tq + e % 2;
      float x = 0.f;
      if (OUT && c < p.vd && k < p.kd)
        x = p.seg_state ? p.seg_state[slot_h * dd + (int64_t)c * p.kd + k] : ld_any(p.init, !p.init_f32, sh * dd + k * p.ik + c * p.ic);
      st[j][e] = x;
    }

  const int Hq = p.H / p.gq, Hk = p.H / p.gk, Hv = p.H / p.gv, Hr = p.r ? p.H / p.gr : 1;
  const int64_t len = run.hi - run.lo;
  const int dir = p.rev ? -1 : 1;
  double total = 0.0;                                          // of the run (warp 0)
  // (chunks lie the same in both directions: a part of one comes first backwards)
  int nv = p.rev ? (int)((len - 1) % L) + 1 : len < L ? (int)len : L;
  for (int64_t c0 = 0; c0 < len; c0 += nv, nv = len - c0 < L ? (int)(len - c0) : L) {
    const int64_t t0 = run.base + (p.rev ? run.hi - 1 - c0 : run.lo + c0);     // token of row 0
    load_tile<MODE, KD, Y::LDK, Y::PK, NT>(sm + Y::K0, p.k, (t0 * Hk + h / p.gk) * p.kd, (int64_t)dir * Hk * p.kd, nv, p.kd);
    {
      const int left = p.vd - cbase;
      load_tile<MODE, Y::VT, Y::LDV, Y::PV, NT>(sm + Y::V0, p.v, (t0 * Hv + h / p.gv) * p.vd + cbase, (int64_t)dir * Hv * p.vd, nv, left);
    }
    if constexpr (OUT) load_tile<MODE, KD, Y::LDK, Y::PK, NT>(sm + Y::Q0, p.q, (t0 * Hq + h / p.gq) * p.kd, (int64_t)dir * Hq * p.kd, nv, p.kd);
    cp_commit();
    if (warp == 0) {
      constexpr int R = L / 32;
      double x[R], sum = 0.0;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = R * lane + i;
        // backwards in time the gate of the token walked before, none for the sequence's last
        const int64_t t = t0 + dir * (int64_t)r + (p.rev ? 1 : 0);
        float gv = 0.f;
        if (r < nv && !(p.rev && t == run.base + run.b)) gv = p.g[t * p.gt + h];
        gv = gv < -200.f ? -200.f : gv;                        // exp of it is 0 either way; -inf would leave inf - inf
        sum += (double)gv * 1.4426950408889634;
        x[i] = sum;
      }
      double inc = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
      }
      // (not inc - sum, which is lost for all of a lane's rows where one gate is not a number)
      const double all = __shfl_sync(0xffffffffu, inc, 31), left = __shfl_up_sync(0xffffffffu, inc, 1), before = lane ? left : 0.0;
      total += all;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const double v = before + x[i];
        const float hi = (float)v;
        lam[R * lane + i] = make_float2(hi, (float)(v - hi));
        wt[R * lane + i] = make_float2(exp2f((float)v), exp2f((float)(all - v)));
      }
    }
    cp_wait<0>();
    __syncthreads();
    const uint32_t uk = sm32(sm + Y::K0), uv = sm32(sm + Y::V0), uq = sm32(sm + Y::Q0), up = sm32(sm + Y::P0);
    if constexpr (OUT) {
      // scores, 16 x 8 at a time: units 0, 1 | 2 .. 5 | 6 .. 11 | 12 .. 19 of row tiles 0 | 1 | 2 | 3
      constexpr int UNITS = (L / 16) * (L / 16 + 1);
      for (int u = warp; u < UNITS; u += NW) {
        const int mi = u < 2 ? 0 : u < 6 ? 1 : u < 12 ? 2 : 3, nt = u - mi * (mi + 1);
        float c[4] = {};
        const uint32_t qa = uq + (mi * 16 + (lane & 15)) * Y::LDK + (lane >> 4) * 16;
        const uint32_t ka = uk + (nt * 8 + (lane & 7)) * Y::LDK + (lane >> 3) * 16;
#pragma unroll 2
        for (int kk = 0; kk < KD / 32; ++kk) {
          uint32_t b[M::NI][4];
#pragma unroll
          for (int s = 0; s < M::NI; ++s) ldsm(b[s], ka + s * Y::PK + kk * 64);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t a[M::NI][4];
#pragma unroll
            for (int s = 0; s < M::NI; ++s) ldsm(a[s], qa + s * Y::PK + kk * 64 + half * 32);
            float y[4] = {};
            float(&z)[4] = M::EXO ? y : c;
#pragma unroll
            for (int t = 2 * M::NI - 2; t >= 0; --t)
#pragma unroll
              for (int i = 0; i < M::NI; ++i)
                if (t - i >= 0 && t - i < M::NI && t <= 2) mma16(z, a[i], b[t - i][2 * half], b[t - i][2 * half + 1]);
            if (M::EXO)
#pragma unroll
              for (int e = 0; e < 4; ++e) c[e] += y[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int i = mi * 16 + gr + 4 * e, j = nt * 8 + 2 * tq;
          const float2 li = lam[i], l0 = lam[j], l1 = lam[j + 1];
          const float x = j <= i ? c[e] * exp2f((li.x - l0.x) + (li.y - l0.y)) : 0.f;
          const float y = j + 1 <= i ? c[e + 1] * exp2f((li.x - l1.x) + (li.y - l1.y)) : 0.f;
          uint32_t s[M::NF];
          planes<M::NF>(x, y, s);
#pragma unroll
          for (int k = 0; k < M::NF; ++k) *reinterpret_cast<uint32_t*>(sm + Y::P0 + k * Y::PP + i * Y::LDP + j * 2) = s[k];
        }
      }
      __syncthreads();
      // outputs, 16 rows at a time
#pragma unroll 1
      for (int mi = 0; mi * 16 < nv; ++mi) {
        float o[2][4] = {};
        const uint32_t qa = uq + (mi * 16 + (lane & 15)) * Y::LDK + (lane >> 4) * 16;
#pragma unroll
        for (int kk = 0; kk < KD / 16; ++kk) {
          uint32_t a[M::NI][4], b[M::NF][4], s0[M::NF], s1[M::NF], s2[M::NF], s3[M::NF];
#pragma unroll
          for (int s = 0; s < M::NI; ++s) ldsm(a[s], qa + s * Y::PK + kk * 32);
          planes<M::NF>(st[2 * kk][0], st[2 * kk][1], s0);
          planes<M::NF>(st[2 * kk + 1][0], st[2 * kk + 1][1], s1);
          planes<M::NF>(st[2 * kk][2], st[2 * kk][3], s2);
          planes<M::NF>(st[2 * kk + 1][2], st[2 * kk + 1][3], s3);
#pragma unroll
          for (int s = 0; s < M::NF; ++s) { b[s][0] = s0[s]; b[s][1] = s1[s]; b[s][2] = s2[s]; b[s][3] = s3[s]; }
          mma_planes<M::NI, M::NF, M::EXO>(o[0], o[1], a, b);
        }
        const int i0 = mi * 16 + gr, i1 = i0 + 8;
        const float w0 = wt[i0].x, w1 = wt[i1].x;
        float keep[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          o[n][0] *= w0; o[n][1] *= w0; o[n][2] *= w1; o[n][3] *= w1;
#pragma unroll
          for (int e = 0; e < 4; ++e) keep[n][e] = o[n][e];
        }
        for (int kj = 0; kj <= mi; ++kj) {
          uint32_t a[M::NF][4], b[M::NI][4];
#pragma unroll
          for (int s = 0; s < M::NF; ++s) ldsm(a[s], up + s * Y::PP + (mi * 16 + (lane & 15)) * Y::LDP + kj * 32 + (lane >> 4) * 16);
          // [token][column] is [k][n]: matrices k 0-7 | k 8-15 of tile 0, then of tile 1
#pragma unroll
          for (int s = 0; s < M::NI; ++s)
            ldsm_t(b[s], uv + s * Y::PV + (kj * 16 + (lane & 15)) * Y::LDV + (warp * 16 + (lane >> 4) * 8) * 2);
          mma_planes<M::NF, M::NI, M::EXO>(o[0], o[1], a, b);
        }
        // A value that is not finite meets the zeros above the diagonal in the product (0 x inf); the recurrence has it at
        // its own token and after only, so what is not finite is summed again over j <= i
        float bad = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) bad = fmaf(o[n][e], 0.f, bad);
        if (bad != 0.f) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(fabsf(o[n][e]) <= 3.402823466e38f)) {
                const int i = mi * 16 + gr + 8 * (e / 2), c = warp * 16 + n * 8 + 2 * tq + e % 2;
                float x = keep[n][e];
#pragma unroll 1
                for (int j = 0; j <= i; ++j)
                  x += sum_planes<M::NF>(sm + Y::P0 + i * Y::LDP + j * 2, Y::PP) * sum_planes<M::NI>(sm + Y::V0 + j * Y::LDV + c * 2, Y::PV);
                o[n][e] = x;
              }
        }
        __syncwarp();
        float dot[2] = {0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = half ? i1 : i0;
          if (i < nv) {
            const int64_t tok = t0 + dir * (int64_t)i;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int c = cw + n * 8 + 2 * tq;
              if (c < p.vd) {
                const float x = o[n][2 * half], y = o[n][2 * half + 1], bx = keep[n][2 * half], by = keep[n][2 * half + 1];
                const int64_t at = (tok * p.H + h) * p.vd + c;
                if (p.out_f32) *reinterpret_cast<float2*>((float*)p.out + at) = make_float2(x, y);
                else *reinterpret_cast<uint32_t*>((bf16*)p.out + at) = pack_bf16x2(x, y);
                if (DOTS && p.r) {
                  const int64_t ra = (tok * Hr + h / p.gr) * p.vd + c;
                  float2 rv;
                  if constexpr (MODE == M_FULL) rv = __ldg((const float2*)((const float*)p.r + ra));
                  else rv = pair_of(__ldg((const unsigned int*)((const bf16*)p.r + ra)));
                  dot[half] = fmaf(bx, rv.x, fmaf(by, rv.y, dot[half]));
                }
              }
            }
          }
        }
        if (DOTS && p.r) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            dot[half] += __shfl_xor_sync(0xffffffffu, dot[half], 1);
            dot[half] += __shfl_xor_sync(0xffffffffu, dot[half], 2);
          }
          if (tq == 0) { rd[warp * L + i0] = dot[0]; rd[warp * L + i1] = dot[1]; }
        }
      }
    }
    // the state: st = exp(lam_L) st + (w V)^T K
    {
      const float all = wt[L - 1].x;
#pragma unroll
      for (int j = 0; j < KT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) st[j][e] *= all;
#pragma unroll 1
      for (int kk = 0; kk * 16 < nv; ++kk) {
        uint32_t a[M::NI][4], wa[M::NU][4];
        // [token][column] is [k][m]
#pragma unroll
        for (int s = 0; s < M::NI; ++s)
          ldsm_t(a[s], uv + s * Y::PV + (kk * 16 + (lane & 7) + ((lane >> 4) & 1) * 8) * Y::LDV + (warp * 16 + ((lane >> 3) & 1) * 8) * 2);
        const int j = kk * 16 + 2 * tq;
        const float w[4] = {wt[j].y, wt[j + 1].y, wt[j + 8].y, wt[j + 9].y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float2 x = pair_of(a[M::NI - 1][e]);
#pragma unroll
          for (int s = M::NI - 2; s >= 0; --s) { const float2 y = pair_of(a[s][e]); x.x += y.x; x.y += y.y; }
          uint32_t z[M::NU];
          planes<M::NU>(x.x * w[e / 2 * 2], x.y * w[e / 2 * 2 + 1], z);
#pragma unroll
          for (int s = 0; s < M::NU; ++s) wa[s][e] = z[s];
        }
#pragma unroll
        for (int nt = 0; nt < KD / 16; ++nt) {
          uint32_t b[M::NI][4];
#pragma unroll
          for (int s = 0; s < M::NI; ++s) ldsm_t(b[s], uk + s * Y::PK + (kk * 16 + (lane & 15)) * Y::LDK + (nt * 16 + (lane >> 4) * 8) * 2);
          mma_planes<M::NU, M::NI, M::EXU>(st[2 * nt], st[2 * nt + 1], wa, b);
        }
      }
    }
    __syncthreads();
    if constexpr (OUT) {
      if (DOTS && p.r && tid < nv) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) x += rd[w * L + tid];
        const int64_t rows = p.cu ? p.T : p.nseq * p.T;
        p.rdot[(vt * rows + t0 + dir * (int64_t)tid) * p.H + h] = x;
      }
    }
  }

  if constexpr (!OUT) {
    if (tid == 0 && vt == 0) p.seg_total[slot_h] = total;
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = cw + gr + 8 * (e / 2), k = 8 * j + 2 * tq + e % 2;
        if (c < p.vd && k < p.kd) p.seg_state[slot_h * dd + (int64_t)c * p.kd + k] = st[j][e];
      }
  } else if ((p.fin || p.fin32) && (p.rev ? run.first : run.last)) {
    float f = 1.f;
    if (p.rev && run.b > run.a) f = expf(p.g[(run.base + run.a) * p.gt + h]);     // the gate of the first token
#pragma unroll
    for (int j = 0; j < KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = cw + gr + 8 * (e / 2), k = 8 * j + 2 * tq + e % 2;
        if (c < p.vd && k < p.kd) {
          const int64_t at = sh * dd + k * p.ik + c * p.ic;
          if (p.fin) st_any(p.fin, !p.fin_f32, at, f * st[j][e]);
          if (p.fin32) p.fin32[at] = f * st[j][e];
        }
      }
  }
}

template <int MODE, int KD, int NW, bool OUT>
int launch_walk(cudaStream_t stream, const Walks& p, int n, const char* name) {
  using Y = Lay<MODE, KD, NW, OUT>;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(walk_kernel<MODE, KD, NW, OUT>, Y::END));
  ProfScope ps(name, stream);
  walk_kernel<MODE, KD, NW, OUT><<<dim3((unsigned)p.w[0].nslots, (unsigned)(p.w[0].H * p.w[0].vt), (unsigned)n), Y::NT, Y::END, stream>>>(p);
  GLA_CHECK_LAUNCH();
  return GLA_OK;
}
template <int MODE, int NW, bool OUT>
int walk_kd(cudaStream_t stream, const Walks& p, int n, const char* name) {
  const int kd = p.w[0].kd;
  if (kd <= 64) return launch_walk<MODE, 64, NW, OUT>(stream, p, n, name);
  if (kd <= 128) return launch_walk<MODE, 128, NW, OUT>(stream, p, n, name);
  return launch_walk<MODE, 256, NW, OUT>(stream, p, n, name);
}
// Blocks of 64 columns where there are no more, of 128 otherwise.  (bf16 heads of up to 128 have walks of their own, so that in the
// bf16 modes columns or features go beyond that.)
static inline int column_tiles(int vd) { return vd <= 64 ? 1 : (vd + 127) / 128; }
template <int MODE, bool OUT>
int walk_nw(cudaStream_t stream, const Walks& p, int n, const char* name) {
  if (p.w[0].vd > 64) return walk_kd<MODE, 8, OUT>(stream, p, n, name);
  if constexpr (MODE == M_FULL) return walk_kd<MODE, 4, OUT>(stream, p, n, name);
  else return launch_walk<MODE, 256, 4, OUT>(stream, p, n, name);
}
// n walks of one kind: the same sizes, runs and column tiles
template <int MODE>
int walk_mode(cudaStream_t stream, Walks p, int n, bool out, const char* name) {
  for (int i = 0; i < n; ++i) p.w[i].vt = column_tiles(p.w[i].vd);
  return out ? walk_nw<MODE, true>(stream, p, n, name) : walk_nw<MODE, false>(stream, p, n, name);
}
int walk_one(cudaStream_t, const Walks&, int n, bool out, const char* name);
int walk_state(cudaStream_t, const Walks&, int n, bool out, const char* name);
int walk_fine(cudaStream_t, const Walks&, int n, bool out, const char* name);
int walk_full(cudaStream_t, const Walks&, int n, bool out, const char* name);

}  // namespace decay
}  // namespace gla
