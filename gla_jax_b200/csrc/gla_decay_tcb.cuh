// The backward walk of decay attention on the fifth-generation tensor cores: dk, dv, the gates' and the first state's gradient,
// 128 tokens at a time, from the sequence's (run's) end.  With dS the gradient of the state that leaves the chunk:
//   ST = K Q^T    DT = V dO^T    IV = K dS    IK = V dS^T                                     (rows j, columns i)
//   P_ji = w_ij ST_ji,  E_ji = w_ij DT_ji  for i >= j        f_j = exp(lam_L - lam_j)
//   dV = f IV + P dO      dK = f IK + E Q      dS <- exp(lam_L) dS + (exp(lam_i) Q)^T dO
// In a chunk of mild gates P and E carry exp(lam_i - lam_L) and the outputs f as they leave; in others IV and IK are multiplied
// in place before P and E, with their whole weights, add to them.
// The scores are formed transposed, so that P and E are where a product takes its left operand from tensor memory, and both
// outputs add up in place.  Tensor memory is full (4 x 128 columns); the sum for dS takes ST's place once P is used.  Shared
// memory holds the four tiles, dS and nothing else: the weighted queries' two planes take the places of V and K, whose
// products are done by then.
//   dg_t = sum over i >= t of (r_i + a_i - c_i - b_i) + <the state that leaves the run, its gradient>
//   M_ji = P_ji DT_ji in float32, r its column and c its row sums;  a = q . (dq from before the chunk), b = k . (dk from behind it)
// from operands in two planes: the sum is over the whole run and its terms cancel.  A value or key
// that is not finite makes it not finite from there back, where dg reads neither: those tokens are summed from the other end,
//   dg_t = <the state that enters the run, its gradient> - sum over i < t of (r_i + a_i - c_i - b_i)
// With the gates' gradient P, E and the image of dS are two bf16 planes, else one (as in the forward).
// Bounded as the forward is: 4 x 4096 tokens of 6 heads, 128 x 128: 77 us; 8191 packed tokens, 16 heads of 128 x 64 with the
// gates' gradient: 177 us; n chunks of 128 x 128: 19 + 9.8 n us, with the gates' gradient 26 + 12.4 n.
#pragma once
#include "gla_decay_tc.cuh"

namespace gla {
namespace decay {

struct TcBack {
  CUtensorMap q, k, v, o;
  Walk w;                                  // k, q, v; H, sizes, gates, runs; seg_state: gradients that enter each run backwards
  const float* a;                          // [TC_COLS][token][H], with gates
  const float *S_runs, *S_end;             // entering states of the runs [slot][H][vd][kd], final states
  const void* S_init;                      // the sequences' first states
  void *dk, *dv;
  int dk_f32;
  float* dg;
};

template <int DK, int DV, bool GATE>
struct BTLay {
  static constexpr int NS = GATE ? 2 : 1;
  static constexpr int TK = DK * 256, TV = DV * 256, SP = DK * DV * 2;
  static constexpr int Q0 = 0, O0 = TK, K0 = O0 + TV, V0 = K0 + TK, H0 = V0 + TV;      // LO is K's place, HI V's if it is large enough
  static constexpr int S0 = H0 + (DV < DK ? TK : 0), STG = S0 + NS * SP;
  static constexpr bool OWN = DK != 128 || DV != 128;                                   // outputs are put together in a place of their own
  static constexpr int G0 = STG + (OWN ? 256 * (DK > DV ? DK : DV) : 0), SUM = G0 + 2 * (int)sizeof(Gates);
  static constexpr int RED = SUM + (GATE ? 2 * 6144 : 0), BAR = RED + 128, USED = BAR + 192 + (DK == 64 ? 16384 : 0);
  static constexpr int END = USED < 120 * 1024 ? 120 * 1024 : USED;
  static constexpr int HI = DV < DK ? H0 : V0, OUT0 = OWN ? STG : S0;
  static_assert(END <= 232448, "shared memory");
  static_assert(DK == DV || 256 * (DK > DV ? DK : DV) >= 4096 * TC_WORK, "a place per warp");
  static_assert(S0 % 1024 == 0 && STG % 1024 == 0, "tiles");
};
enum TbBar { C_LOAD = 0, C_ST = 1, C_I = 2, C_DV = 3, C_U = 4, C_P = 5, C_W = 6, C_S = 7, C_G = 8, C_GFREE = 10, C_E = 12, C_COUNT = 14, C_TMEM = 14, C_ODD = 15, C_BACK = 16 };

// o (a row of tensor memory, D / TC_COLS columns from the worker's first) += sum over i >= row of P_i V_i, for a chunk in which V holds
// something that is not finite (see masked_sums)
template <int D, int NP>
__device__ __noinline__ void masked_add(uint32_t tp, uint32_t to, uint32_t tv, int row, int qt) {
#pragma unroll 1
  for (int c0 = qt * (D / TC_COLS); c0 < (qt + 1) * (D / TC_COLS); c0 += 16) {
    uint32_t r[16];
    __syncwarp();
    tmem_ld16(to + c0, r);
    tmem_ld_wait();
#pragma unroll 1
    for (int k = 0; k < 8; ++k) {
      float p[16];
      __syncwarp();
      load_scores<NP>(tp + score_at<NP>(k), p);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int t = 16 * k + j;
        const float pj = p[j];
        const uint32_t at = tv + (c0 >> 6) * 16384;
        const uint4 a = lds16(at + sw128_chunk(t, (c0 >> 3) & 7)), b = lds16(at + sw128_chunk(t, ((c0 >> 3) & 7) + 1));
        const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (t >= row)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 v = pair_of(u[e]);
            r[2 * e] = __float_as_uint(fmaf(pj, v.x, __uint_as_float(r[2 * e])));
            r[2 * e + 1] = __float_as_uint(fmaf(pj, v.y, __uint_as_float(r[2 * e + 1])));
          }
      }
    }
    __syncwarp();
    tmem_st16(to + c0, r);
  }
  tmem_st_wait();
}
// Rows of a tile times exp(lam_i) in two planes, from one place to two others.
template <int D>
__device__ __forceinline__ void weigh_to(uint32_t tile, uint32_t hi, uint32_t lo, const float2* wt) {
  const int r0 = threadIdx.x / 8, c = threadIdx.x % 8;
  const uint32_t at0 = sw128_chunk(r0, c);
#pragma unroll 2
  for (int j = 0; j < 128 / TC_ROWS; ++j) {
    const float w = wt[r0 + TC_ROWS * j].x;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint32_t at = b * 16384 + j * TC_ROWS * 128 + at0;
      const uint4 x = lds16(tile + at);
      const uint32_t u[4] = {x.x, x.y, x.z, x.w};
      uint32_t s[4][2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = pair_of(u[e]);
        planes<2>(y.x * w, y.y * w, s[e]);
      }
      sts16(hi + at, make_uint4(s[0][0], s[1][0], s[2][0], s[3][0]));
      sts16(lo + at, make_uint4(s[0][1], s[1][1], s[2][1], s[3][1]));
    }
  }
}
__device__ __forceinline__ bool workers_or(bool x) {          // barrier of the workers, and whether any has x
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
               : "=r"(r) : "r"((uint32_t)x), "n"(TC_WORK * 32) : "memory");
  return r != 0;
}
// 16 values of each of 32 lanes summed over the lanes: lane l is left with the sum of value l % 16
__device__ __forceinline__ float lane_sums(float (&v)[16], int lane) {
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], 16);
#pragma unroll
  for (int s = 8; s; s >>= 1)
#pragma unroll
    for (int j = 0; j < s; ++j) {
      const float give = (lane & s) ? v[j] : v[j + s], keep = (lane & s) ? v[j + s] : v[j];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, give, s);
    }
  return v[0];
}

template <int DK, int DV, bool GATE>
__global__ void __launch_bounds__(TC_THREADS, 1) tc_back_kernel(const __grid_constant__ TcBack a) {
  using Y = BTLay<DK, DV, GATE>;
  constexpr int NS = Y::NS, HV = DV / TC_COLS, HK = DK / TC_COLS;
  const Walk& p = a.w;
  extern __shared__ __align__(1024) uint8_t sm[];
  Gates* gates = reinterpret_cast<Gates*>(sm + Y::G0);
  float* sums = reinterpret_cast<float*>(sm + Y::SUM);          // [2][12][128]: r by row group, c and b by half
  double* red = reinterpret_cast<double*>(sm + Y::RED);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int h = blockIdx.y;
  grid_dep_wait();
  grid_dep_launch();
  const Run run = find_run(p, blockIdx.x);
  if (run.zlo < run.zhi) {
    for (int64_t i = tid; i < (run.zhi - run.zlo) * p.kd; i += TC_THREADS) st_any(a.dk, !a.dk_f32, ((run.zlo + i / p.kd) * p.H + h) * p.kd + i % p.kd, 0.f);
    for (int64_t i = tid; i < (run.zhi - run.zlo) * p.vd; i += TC_THREADS) st_any(a.dv, 1, ((run.zlo + i / p.vd) * p.H + h) * p.vd + i % p.vd, 0.f);
    if (GATE)
      for (int64_t i = tid; i < run.zhi - run.zlo; i += TC_THREADS) a.dg[(run.zlo + i) * p.H + h] = 0.f;
  }
  if (!run.any) return;
  const uint32_t base = smem_u32(sm), bars = base + Y::BAR;
  const auto bar = [&](int b) { return bars + 8 * b; };
  if (tid == 0) {
    for (int i = 0; i < C_COUNT; ++i) mbar_init(bar(i), i == C_P || i == C_W || i == C_S || i >= C_GFREE ? TC_WORK : 1);
    asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(bar(C_ODD)), "r"(0) : "memory");
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(bar(C_TMEM), 512);
    tmem_relinquish();
  }
  const int64_t sh = run.s * p.H + h, dd = (int64_t)p.kd * p.vd, slot_h = (int64_t)blockIdx.x * p.H + h;
  const int len = (int)(run.hi - run.lo), chunks = (len + 127) / 128;
  const int64_t r0 = run.base + run.lo, rows = p.cu ? p.T : p.nseq * p.T;
  const auto rows_of = [&](int i) { const int c0 = 128 * (chunks - 1 - i); return len - c0 < 128 ? len - c0 : 128; };   // step i: from the end
  const auto token = [&](int i) { return r0 + 128 * (chunks - 1 - i); };

  const int q4 = warp & 3, qt = (warp >> 2) % TC_COLS, row = 32 * q4 + lane;      // (workers)
  const uint32_t lane_base = (uint32_t)(32 * q4) << 16;
  float S[HV];                                                               // dS: row `row`, columns HV qt + [0, HV)
  const int cols = row < p.kd ? p.vd - HV * qt : 0;
  if (warp < TC_WORK) {
    double dot = 0.0;
    const int64_t at = sh * dd + (int64_t)row * p.vd + HV * qt, across = row + (int64_t)HV * qt * p.kd;      // [feature][column], [column][feature]
    if (p.seg_state) {
      const float* x = p.seg_state + slot_h * dd + across;
#pragma unroll
      for (int j = 0; j < HV; ++j) S[j] = j < cols ? x[(int64_t)j * p.kd] : 0.f;
    } else {
      load_side<HV>(S, p.init_f32 ? (const void*)((const float*)p.init + at) : (const void*)((const bf16*)p.init + at), p.init_f32, cols);
    }
    if (GATE) {
      // with the state that leaves the run
      float x[HV];
      if (run.last) {
        load_side<HV>(x, a.S_end + at, 1, cols);
      } else {
        const float* y = a.S_runs + (slot_h + p.H) * dd + across;
#pragma unroll
        for (int j = 0; j < HV; ++j) x[j] = j < cols ? y[(int64_t)j * p.kd] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < HV; ++j) dot += (double)S[j] * x[j];
    }
    if (GATE) {
#pragma unroll
      for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      if (lane == 0) red[warp] = dot;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(bar(C_TMEM)));
  const uint32_t tST = tmem, tDT = tmem + 128, tIV = tmem + 256, tIK = tmem + 384;
  bool ok = true;

  if (warp == TC_WORK) {
    // ================= products =================
    if (lane == 0) {
      const auto kcol = [](int s) { return (uint32_t)((s >> 2) * 16384 + (s & 3) * 32); };
      const uint64_t kQ = desc_kmajor(base + Y::Q0, 16384, 0), kO = desc_kmajor(base + Y::O0, 16384, 0), kK = desc_kmajor(base + Y::K0, 16384, 0),
                     kV = desc_kmajor(base + Y::V0, 16384, 0), mQ = desc_mnmajor(base + Y::Q0, 16384, 0), mO = desc_mnmajor(base + Y::O0, 16384, 0),
                     mS = desc_mnmajor(base + Y::S0, DK * 128, 0), kS = desc_kmajor(base + Y::S0, DK * 128, 0),
                     mH = desc_mnmajor(base + Y::HI, 16384, 0), mL = desc_mnmajor(base + Y::K0, 16384, 0);
      for (int i = 0; i < chunks; ++i) {
        const uint32_t ph = i & 1;
        wait_for(ok, bar(C_LOAD), ph);
        wait_for(ok, bar(C_S), ph);                // dS's image; everything of the step before is read
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < DK / 16; ++s) umma_bf16(tST, desc_advance(kK, kcol(s)), desc_advance(kQ, kcol(s)), idesc_bf16(128, 128, 0, 0), s > 0);
#pragma unroll
        for (int s = 0; s < DV / 16; ++s) umma_bf16(tDT, desc_advance(kV, kcol(s)), desc_advance(kO, kcol(s)), idesc_bf16(128, 128, 0, 0), s > 0);
        umma_commit(bar(C_ST));
#pragma unroll
        for (int n = NS - 1; n >= 0; --n)
#pragma unroll
          for (int s = 0; s < DK / 16; ++s)
            umma_bf16(tIV, desc_advance(kK, kcol(s)), desc_advance(mS, n * Y::SP + s * 2048), idesc_bf16(128, DV, 0, 1), n < NS - 1 || s > 0);
#pragma unroll
        for (int n = NS - 1; n >= 0; --n)
#pragma unroll
          for (int s = 0; s < DV / 16; ++s)
            umma_bf16(tIK, desc_advance(kV, kcol(s)), desc_advance(kS, n * Y::SP + (s >> 2) * DK * 128 + (s & 3) * 32), idesc_bf16(128, DK, 0, 0),
                      n < NS - 1 || s > 0);
        umma_commit(bar(C_I));
        wait_for(ok, bar(C_P), ph);
        tc_fence_after();
        uint32_t odd;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(odd) : "r"(bar(C_ODD) + 4 * (i & 1)) : "memory");
        if (odd != (uint32_t)(i + 1)) {
#pragma unroll
          for (int s = 0; s < 8 * NS; ++s) umma_ts(tIV, tST + score_at<NS>(s & 7) + 8 * (s >> 3), desc_advance(mO, (s & 7) * 2048), idesc_bf16(128, DV, 0, 1), 1);
#pragma unroll
          for (int s = 0; s < 8 * NS; ++s) umma_ts(tIK, tDT + score_at<NS>(s & 7) + 8 * (s >> 3), desc_advance(mQ, (s & 7) * 2048), idesc_bf16(128, DK, 0, 1), 1);
        }
        umma_commit(bar(C_DV));
        wait_for(ok, bar(C_W), ph);
        tc_fence_after();
#pragma unroll
        for (int n = 1; n >= 0; --n)
#pragma unroll
          for (int s = 0; s < 8; ++s)
            umma_bf16(tST, desc_advance(n ? mL : mH, s * 2048), desc_advance(mO, s * 2048), idesc_bf16(128, DV, 1, 1), n < 1 || s > 0);
        umma_commit(bar(C_U));
      }
    }
    __syncwarp();
  } else if (warp == TC_WORK + 1) {
    // ================= tensor copies =================
    if (lane == 0) {
      const int hk = h / p.gq;
      for (int i = 0; i < chunks; ++i) {
        const int z = (int)token(i);
        if (i >= 1) wait_for(ok, bar(C_U), (i - 1) & 1);
        mbar_arrive_expect_tx(bar(C_LOAD), 2 * (Y::TK + Y::TV));
        for (int b = 0; b < DK / 64; ++b) {
          tma_load_3d(base + Y::K0 + b * 16384, &a.k, 64 * b, hk, z, bar(C_LOAD));
          tma_load_3d(base + Y::Q0 + b * 16384, &a.q, 64 * b, hk, z, bar(C_LOAD));
        }
        for (int b = 0; b < DV / 64; ++b) {
          tma_load_3d(base + Y::V0 + b * 16384, &a.v, 64 * b, h, z, bar(C_LOAD));
          tma_load_3d(base + Y::O0 + b * 16384, &a.o, 64 * b, h, z, bar(C_LOAD));
        }
      }
    }
    __syncwarp();
  } else if (warp == TC_WORK + 2) {
    // ================= gates, and their gradient a step behind =================
    double carry = 0.0;
    int back = 0;                                // tokens from the run's first on whose sum is not finite; their dg holds the term
    if (GATE)
      for (int w = 0; w < TC_WORK; ++w) carry += red[w];
    const auto gradient = [&](int i) {
      const int nv = rows_of(i);
      const int64_t t0 = token(i);
      const float* s = sums + (i & 1) * 1536;
      wait_for(ok, bar(C_E + (i & 1)), (i >> 1) & 1);
      double e[4], sum = 0.0;
      float own[4];
#pragma unroll
      for (int u = 3; u >= 0; --u) {
        const int t = 4 * lane + u;
        double x = 0.0;
        if (t < nv) {
          const float* y = s + t;
#pragma unroll
          for (int m = 0; m < 4; ++m) x += (double)y[128 * m];
#pragma unroll
          for (int m = 0; m < TC_COLS; ++m) x += (double)a.a[(m * rows + t0 + t) * p.H + h] - (double)y[512 + 128 * m] - (double)y[1024 + 128 * m];
        }
        sum += x;
        e[u] = sum;
        own[u] = (float)x;
      }
      double inc = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_down_sync(0xffffffffu, inc, d);
        if (lane + d < 32) inc += y;
      }
      // (what is behind this lane's tokens; not inc - sum, which is lost where sum is not finite)
      const double next = __shfl_down_sync(0xffffffffu, inc, 1), behind = carry + (lane < 31 ? next : 0.0);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (4 * lane + u < nv) {
          const double y = behind + e[u];
          a.dg[(t0 + 4 * lane + u) * p.H + h] = isfinite(y) ? (float)y : own[u];
          if (!isfinite(y)) back = max(back, (int)(t0 - r0) + 4 * lane + u + 1);
        }
      carry += __shfl_sync(0xffffffffu, inc, 0);
    };
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
    if (chunks) g = gates_of(p, token(0), rows_of(0), h, lane);
    for (int i = 0; i < chunks; ++i) {
      if (GATE && i >= 2) gradient(i - 2);
      if (i >= 2) wait_for(ok, bar(C_GFREE + (i & 1)), ((i - 2) >> 1) & 1);
      if (p.gt != 0 || i < 2 || rows_of(i) != rows_of(i - 2)) scan_gates(g, gates[i & 1], lane);      // (as in the forward)
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C_G + (i & 1)));
      if (i + 1 < chunks) g = gates_of(p, token(i + 1), rows_of(i + 1), h, lane);
    }
    if (GATE)
      for (int i = chunks >= 2 ? chunks - 2 : 0; i < chunks; ++i) gradient(i);
    if (GATE) {
      back = __reduce_max_sync(0xffffffffu, back);
      if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(bar(C_BACK)), "r"(back) : "memory");
    }
  } else {
    // ================= workers =================
    const auto put_state = [&]() {
      if (row < DK) {
#pragma unroll
        for (int j = 0; j < HV; j += 8) {
          uint32_t s[4][NS];
#pragma unroll
          for (int e = 0; e < 4; ++e) planes<NS>(S[j + 2 * e], S[j + 2 * e + 1], s[e]);
          const int c8 = (HV * qt + j) / 8;
#pragma unroll
          for (int k = 0; k < NS; ++k)
            sts16(base + Y::S0 + k * Y::SP + (c8 >> 3) * DK * 128 + sw128_chunk(row, c8 & 7), make_uint4(s[0][k], s[1][k], s[2][k], s[3][k]));
        }
      }
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C_S));
    };
    put_state();
    for (int i = 0; i < chunks; ++i) {
      const int nv = rows_of(i);
      const int64_t t0 = token(i);
      const uint32_t ph = i & 1;
      const Gates& gs = gates[i & 1];
      float* sum = sums + (i & 1) * 1536;
      if (!all_done(bar(C_G + (i & 1)), (i >> 1) & 1, bar(C_LOAD), ph, bar(C_ST), ph)) {
        wait_for(ok, bar(C_G + (i & 1)), (i >> 1) & 1);
        wait_for(ok, bar(C_LOAD), ph);
        wait_for(ok, bar(C_ST), ph);
      }
      tc_fence_after();
      const bool mild = gs.reach <= MILD;
      const float wj = gs.wt[row].y;
      float rowsum = 0.f;
#pragma unroll 1
      for (int sb = qt * (8 / TC_COLS); sb < (qt + 1) * (8 / TC_COLS); ++sb) {
        const int grp = sb >> 1;             // columns (tokens i) 16 sb + [0, 16), of the group of 32
        uint32_t pk[8 * NS], ek[8 * NS];
        if (grp < q4) {
#pragma unroll
          for (int e = 0; e < 8 * NS; ++e) pk[e] = ek[e] = 0u;
          if (GATE && lane < 16) sum[128 * q4 + 16 * sb + lane] = 0.f;
        } else {
          uint32_t x[16], y[16];
          float m[GATE ? 16 : 1];
          tmem_ld16(tST + lane_base + 16 * sb, x);
          tmem_ld16(tDT + lane_base + 16 * sb, y);
          tmem_ld_wait();
          const bool own = grp == q4, sharp = !mild && own && !(gs.span[q4] <= 80.f);
          const float cf = mild ? 1.f : own ? gs.cd[row] : gs.cf[grp - 1][row];
          const float* rf = mild ? gs.up : gs.rf;
          const float2 lj = gs.lam[row];
          const int first = own ? lane - 16 * (sb & 1) : 0, end = nv - 16 * sb;           // columns that count
          const float wm = mild ? wj : 1.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float s[2], d[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int c = 2 * e + u;
              const float w = sharp ? decay_of(gs.lam[16 * sb + c], lj) : rf[16 * sb + c] * cf;
              const bool in = c >= first && c < end;
              s[u] = in ? __uint_as_float(x[c]) * w : 0.f;
              d[u] = in ? __uint_as_float(y[c]) * w : 0.f;
              if constexpr (GATE) {
                m[c] = in ? s[u] * wm * __uint_as_float(y[c]) : 0.f;      // (s alone may be near the top)
                rowsum += m[c];
              }
            }
            set_scores<NS>(pk, e, s[0], s[1]);
            set_scores<NS>(ek, e, d[0], d[1]);
          }
          if constexpr (GATE) {
            const float t = lane_sums(m, lane);
            if (lane < 16) sum[128 * q4 + 16 * sb + lane] = t;
          }
        }
        store_scores<NS>(tST + lane_base + score_at<NS>(sb), pk);
        store_scores<NS>(tDT + lane_base + score_at<NS>(sb), ek);
      }
      if (GATE) sum[512 + 128 * qt + row] = rowsum;
      bool odd = check_rows<DV>(base + Y::O0, nv);
      odd = check_rows<DK>(base + Y::Q0, nv) || odd;
      wait_for(ok, bar(C_I), ph);
      tc_fence_after();
      float dot = 0.f;
      if (!mild) {
#pragma unroll 1
        for (int c0 = 0; c0 < HV; c0 += 16) {
          uint32_t x[16];
          tmem_ld16(tIV + lane_base + HV * qt + c0, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(wj * __uint_as_float(x[e]));
          tmem_st16(tIV + lane_base + HV * qt + c0, x);
        }
      }
      if (!mild || GATE)
#pragma unroll 1
      for (int c0 = 0; c0 < HK; c0 += 16) {
        uint32_t x[16];
        tmem_ld16(tIK + lane_base + HK * qt + c0, x);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(wj * __uint_as_float(x[e]));
        if (!mild) tmem_st16(tIK + lane_base + HK * qt + c0, x);
        if constexpr (GATE) {
          const int c8 = (HK * qt + c0) / 8;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint4 k = lds16(base + Y::K0 + (c8 >> 3) * 16384 + sw128_chunk(row, (c8 & 7) + b));
            const uint32_t u[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 z = pair_of(u[e]);
              dot = fmaf(__uint_as_float(x[8 * b + 2 * e]), z.x, fmaf(__uint_as_float(x[8 * b + 2 * e + 1]), z.y, dot));
            }
          }
        }
      }
      if (GATE) sum[1024 + 128 * qt + row] = dot;
      tmem_st_wait();
      fence_async_smem();
      tc_fence_before();
      odd = workers_or(odd);              // (and K and V are done with)
      if (odd) {
        tc_fence_after();
        masked_add<DV, NS>(tST + lane_base, tIV + lane_base, base + Y::O0, row, qt);
        masked_add<DK, NS>(tDT + lane_base, tIK + lane_base, base + Y::Q0, row, qt);
        tc_fence_before();
        if (tid == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(bar(C_ODD) + 4 * (i & 1)), "r"(i + 1) : "memory");
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(C_P));
        if (GATE) mbar_arrive(bar(C_E + (i & 1)));
      }
      weigh_to<DK>(base + Y::Q0, base + Y::HI, base + Y::K0, gs.wt);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C_W));
      wait_for(ok, bar(C_DV), ph);
      tc_fence_after();
      // the outputs, as in the forward
      const auto leave = [&](auto is_dk) {
        constexpr bool DKO = decltype(is_dk)::value;
        constexpr int HD = DKO ? HK : HV;
        const int nd = DKO ? p.kd : p.vd;
        const uint32_t t = (DKO ? tIK : tIV) + lane_base + HD * qt;
        // a warp's place must be its own for dv and dk both: with equal sizes that is its part of the rows, else 4 KB of their own
        const auto place = [&](int r, int c) {             // of piece c of row r of the warp
          const int c8 = HD / 8 * qt + c;
          return base + Y::OUT0 + (DK == DV ? (c8 >> 3) * 16384 + sw128_chunk(32 * q4 + r, c8 & 7) : 4096 * warp + sw128_chunk(r, c));
        };
        const float f = mild ? wj : 1.f;
        if (DKO && a.dk_f32) {
          float* o = (float*)a.dk + ((t0 + row) * p.H + h) * nd + HD * qt;
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 16) {
            uint32_t x[16];
            tmem_ld16(t + c0, x);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (row < nv && HD * qt + c0 + e < nd)
                *reinterpret_cast<float4*>(o + c0 + e) = make_float4(f * __uint_as_float(x[e]), f * __uint_as_float(x[e + 1]), f * __uint_as_float(x[e + 2]), f * __uint_as_float(x[e + 3]));
          }
          return;
        }
#pragma unroll 2
        for (int c0 = 0; c0 < HD; c0 += 16) {
          uint32_t x[16], w[8];
          tmem_ld16(t + c0, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(f * __uint_as_float(x[2 * e]), f * __uint_as_float(x[2 * e + 1]));
          sts16(place(lane, c0 / 8), make_uint4(w[0], w[1], w[2], w[3]));
          sts16(place(lane, c0 / 8 + 1), make_uint4(w[4], w[5], w[6], w[7]));
        }
        constexpr int LR = HD / 8, RI = 32 / LR;
        __syncwarp();
        const int c8 = HD / 8 * qt + lane % LR;
        bf16* o = (bf16*)(DKO ? a.dk : a.dv) + ((t0 + 32 * q4 + lane / LR) * p.H + h) * nd + 8 * c8;
#pragma unroll
        for (int j = 0; j < 32; j += RI) {
          const int r = j + lane / LR;
          if (32 * q4 + r < nv && 8 * c8 < nd) *reinterpret_cast<uint4*>(o) = lds16(place(r, lane % LR));
          o += (int64_t)RI * p.H * nd;
        }
        __syncwarp();
      };
      leave(std::false_type());
      leave(std::true_type());
      wait_for(ok, bar(C_U), ph);
      tc_fence_after();
      const float all = gs.wt[127].x;
#pragma unroll
      for (int c0 = 0; c0 < HV; c0 += 16) {
        uint32_t u[16];
        tmem_ld16(tST + lane_base + HV * qt + c0, u);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) S[c0 + e] = fmaf(all, S[c0 + e], __uint_as_float(u[e]));
      }
      if (i + 1 < chunks) put_state();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C_GFREE + (i & 1)));
    }
    if (p.fin && run.first) {
      const int64_t at = sh * dd + (int64_t)row * p.vd + HV * qt;
      store_side<HV>(S, p.fin_f32 ? (void*)((float*)p.fin + at) : (void*)((bf16*)p.fin + at), p.fin_f32, cols);
    }
  }
  if (!ok && lane == 0) atomicAdd(&g_wait_timeouts, 1u);
  tc_fence_before();
  __syncthreads();
  if constexpr (GATE) {
    int back;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(back) : "r"(bar(C_BACK)) : "memory");
    if (back) {
      // from the run's first token on, with the state that enters the run (S is its gradient)
      if (warp < TC_WORK) {
        double dot = 0.0;
        const int64_t at = sh * dd + (int64_t)row * p.vd + HV * qt;
        const float* y = a.S_runs + slot_h * dd + row + (int64_t)HV * qt * p.kd;
#pragma unroll
        for (int j = 0; j < HV; ++j)
          if (j < cols) dot += (double)S[j] * (run.first ? ld_any(a.S_init, !p.init_f32, at + j) : y[(int64_t)j * p.kd]);
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (lane == 0) red[warp] = dot;
      }
      __syncthreads();
      if (warp == TC_WORK + 2) {
        double dot = 0.0;
        for (int w = 0; w < TC_WORK; ++w) dot += red[w];
        for (int t0 = 0; t0 < back; t0 += 32) {
          float* at = a.dg + (r0 + t0 + lane) * p.H + h;
          const double x = t0 + lane < back ? (double)*at : 0.0;
          double inc = x;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
          }
          // (what is before this lane's token; not inc - x, which is lost where x is not finite)
          const double prev = __shfl_up_sync(0xffffffffu, inc, 1);
          if (t0 + lane < back) *at = (float)(dot - (lane ? prev : 0.0));
          dot -= __shfl_sync(0xffffffffu, inc, 31);
        }
      }
    }
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int DK, int DV, bool GATE>
int launch_tc_back(cudaStream_t stream, TcBack& b, const void* dout) {
  using Y = BTLay<DK, DV, GATE>;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(tc_back_kernel<DK, DV, GATE>, Y::END));
  const Walk& p = b.w;
  const int64_t rows = p.cu ? p.T : p.nseq * p.T;
  GLA_TRY(make_map_tokens(&b.q, p.q, rows, p.H / p.gq, p.kd));
  GLA_TRY(make_map_tokens(&b.k, p.k, rows, p.H / p.gq, p.kd));
  GLA_TRY(make_map_tokens(&b.v, p.v, rows, p.H, p.vd));
  GLA_TRY(make_map_tokens(&b.o, dout, rows, p.H, p.vd));
  ProfScope ps("decay_back_kernel", stream);
  GLA_LAUNCHED(launch_overlapped(tc_back_kernel<DK, DV, GATE>, dim3((unsigned)p.nslots, (unsigned)p.H), dim3(TC_THREADS), Y::END, stream, b));
  return GLA_OK;
}

}  // namespace decay
}  // namespace gla
