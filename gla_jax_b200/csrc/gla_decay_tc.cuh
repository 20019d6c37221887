// The walks of gla_decay.cuh on the fifth-generation tensor cores: bf16, head sizes up to 128, 128 tokens at a time.
//
// Per chunk, one thread issues  SC = Q K^T,  OI = Q S,  OA = P V  and  U = (w K)^T V  (w = exp(lam_L - lam_j), in two or three
// bf16 planes); 256 threads turn SC into P in tensor memory (a thread per row and half of the columns), weigh K in place, add
// exp(lam_i) OI + OA into out, and keep the state in registers: S <- exp(lam_L) S + U, from where its bf16 image goes to
// shared memory for the next chunk.
//
// Why.  The same walk in mma.sync spends 14,000 instructions per 64 tokens, of which 1900 multiply: operand fragments, their
// conversion and the accumulators' addressing are the work.  Here operands go from shared memory to the tensor cores as the
// copies left them, and a chunk of 128 takes about 1500 instructions in each of eight warps.
//
// Tiles: 128 rows x 64 columns of bf16, 128-byte rows, 16-byte pieces at piece ^ (row % 8) (tc_ptx.cuh); D columns are D / 64
// of them.  Copies are cp.async rather than tensor copies, because a sequence may start and end anywhere: rows past its end
// are zeros.
#pragma once
#include "gla_decay.cuh"

namespace gla {
namespace decay {

using namespace tc;

__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
         "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (+)= A[tensor memory] B[shared memory]
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float ex2(float x) {      // 2^-22 relative, 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

static __device__ unsigned int g_wait_timeouts = 0;
static inline unsigned int read_wait_timeouts() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_wait_timeouts, sizeof(v));
  return v;
}

// 128 rows of D columns into D / 64 tiles; src: row 0.  Rows from nv on and columns from d on are zeros.
template <int D>
__device__ __forceinline__ void fetch128(uint32_t tile, const bf16* src, int64_t step, int nv, int d) {
  constexpr int C8 = D / 8, RS = 256 / C8;
  const int r0 = threadIdx.x / C8, c = threadIdx.x % C8;
  const bf16* g = src + r0 * step + c * 8;
  const uint32_t dst = tile + (c >> 3) * 16384 + sw128_chunk(r0, c & 7);
  const int n = c * 8 < d ? nv - r0 : 0;
#pragma unroll 2
  for (int j = 0; j < 128 / RS; ++j) {
    cp16(dst + j * RS * 128, RS * j < n ? g : src, RS * j < n);
    g += RS * step;
  }
}

// What a chunk of 128 needs of its gates, made by one warp, four rows a lane.  lam: running sums, base 2, as two floats;
// wt: exp(lam_i), exp(lam_L - lam_i).  The weight exp(lam_i - lam_j) of a pair in different groups of 32 rows is rf_i cf_j over
// the last token before i's group (384 exponentials for 12288 pairs), inside a group it is formed as it stands.
struct Gates {
  float2 lam[128], wt[128];
  float rf[128], cf[3][128];           // cf[g - 1]: to the last token before row group g
};
__device__ __forceinline__ float4 gates_of(const Walk& p, int64_t t0, int nv, int h, int lane) {
  float g[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) g[i] = 4 * lane + i < nv ? p.g[(t0 + 4 * lane + i) * p.gt + h] : 0.f;
  return make_float4(g[0], g[1], g[2], g[3]);
}
__device__ __forceinline__ double scan_gates(float4 g, Gates& s, int lane) {
  const float x[4] = {g.x, g.y, g.z, g.w};
  double v[4], sum = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // exp of less than -200 is 0 either way; -inf would leave inf - inf
    sum += (double)(x[i] < -200.f ? -200.f : x[i]) * 1.4426950408889634;
    v[i] = sum;
  }
  double inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  const double all = __shfl_sync(0xffffffffu, inc, 31), before = inc - sum;
  const double at[3] = {__shfl_sync(0xffffffffu, inc, 7), __shfl_sync(0xffffffffu, inc, 15), __shfl_sync(0xffffffffu, inc, 23)};
  const double own = lane < 8 ? 0.0 : lane < 16 ? at[0] : lane < 24 ? at[1] : at[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double y = before + v[i];
    const float hi = (float)y;
    const int r = 4 * lane + i;
    s.lam[r] = make_float2(hi, (float)(y - hi));
    s.wt[r] = make_float2(ex2(hi), ex2((float)(all - y)));
    s.rf[r] = ex2((float)(y - own));
#pragma unroll
    for (int m = 0; m < 3; ++m)
      if (lane < 8 * (m + 1)) s.cf[m][r] = ex2((float)(at[m] - y));
  }
  return all;
}
__device__ __forceinline__ float decay_of(float2 i, float2 j) { return ex2((i.x - j.x) + (i.y - j.y)); }

// Rows of a tile times a weight per row, in NU planes: the first in place, the others at lo, lo + plane, ...
template <int D, int NU>
__device__ __forceinline__ void weigh(uint32_t tile, uint32_t lo, uint32_t plane, const float2* wt, bool rev) {
  const int r0 = threadIdx.x / 8, c = threadIdx.x % 8;
  const float* w_ = &wt[r0].x + (rev ? 0 : 1);
  const uint32_t at0 = sw128_chunk(r0, c);
#pragma unroll 1
  for (int j = 0; j < 4; ++j) {
    const float w = w_[64 * j];
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint32_t at = b * 16384 + j * 4096 + at0;
      const uint4 x = lds16(tile + at);
      const uint32_t u[4] = {x.x, x.y, x.z, x.w};
      uint32_t s[4][NU];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = pair_of(u[e]);
        planes<NU>(y.x * w, y.y * w, s[e]);
      }
      sts16(tile + at, make_uint4(s[0][0], s[1][0], s[2][0], s[3][0]));
#pragma unroll
      for (int k = 1; k < NU; ++k) sts16(lo + (k - 1) * plane + at, make_uint4(s[0][k], s[1][k], s[2][k], s[3][k]));
    }
  }
}
// whether the pieces that the thread itself fetched of a tile hold something that is not finite
template <int D>
__device__ __forceinline__ bool odd_values(uint32_t tile) {
  constexpr int C8 = D / 8, RS = 256 / C8;
  const int r0 = threadIdx.x / C8, c = threadIdx.x % C8;
  bool x = false;
#pragma unroll 2
  for (int j = 0; j < 128 / RS; ++j) {
    const uint4 v = lds16(tile + (c >> 3) * 16384 + sw128_chunk(r0, c & 7) + j * RS * 128);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x = x || (u[e] & 0x7f80u) == 0x7f80u || (u[e] & 0x7f800000u) == 0x7f800000u;
  }
  return x;
}
// What is not finite in OA = P V, by sums over the tokens up to the row's own (UP = false) or from it on (UP): in the product,
// zeros of P meet what is not finite in V, and 0 x inf is not a number, where the recurrence has it at its own token and after
// (before) only.
// P: this lane's row in tensor memory; 16 columns at a time.
template <int DV, bool UP>
__device__ __noinline__ void masked_sums(uint32_t tp, uint32_t to, uint32_t tv, int row, int half) {
#pragma unroll 1
  for (int c0 = half * (DV / 2); c0 < (half + 1) * (DV / 2); c0 += 16) {
    float o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll 1
    for (int k = 0; k < 8; ++k) {
      uint32_t pk[8];
      __syncwarp();
      tmem_ld8(tp + 64 * (k >> 2) + 8 * (k & 3), pk);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int t = 16 * k + j;
        const float2 y = pair_of(pk[j / 2]);
        const float pj = j % 2 ? y.y : y.x;
        const uint32_t at = tv + (c0 >> 6) * 16384;
        const uint4 a = lds16(at + sw128_chunk(t, (c0 >> 3) & 7)), b = lds16(at + sw128_chunk(t, ((c0 >> 3) & 7) + 1));
        const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (UP ? t >= row : t <= row)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 v = pair_of(u[e]);
            o[2 * e] = fmaf(pj, v.x, o[2 * e]);
            o[2 * e + 1] = fmaf(pj, v.y, o[2 * e + 1]);
          }
      }
    }
    uint32_t r[16];
    __syncwarp();
    tmem_ld16(to + c0, r);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (!(fabsf(__uint_as_float(r[e])) <= 3.402823466e38f)) r[e] = __float_as_uint(o[e]);
    tmem_st16(to + c0, r);
  }
  tmem_st_wait();
}

template <int DK, int DV, int NU, int NS, bool OUT>
struct TLay {
  static constexpr int NK = OUT && NU + NS <= 3 ? 2 : 1;                  // stages of K
  static constexpr int TK = DK * 256, TV = DV * 256, SP = DK * DV * 2;
  static constexpr int Q0 = 0, K0 = Q0 + (OUT ? TK : 0), V0 = K0 + NK * TK, L0 = V0 + TV, S0 = L0 + (NU - 1) * TK;
  static constexpr int G0 = S0 + (OUT ? NS * SP : 0), BAR = G0 + 2 * (int)sizeof(Gates), USED = BAR + 64;
  // one block per SM, whatever the sizes: each takes all of the tensor memory
  static constexpr int END = USED < 120 * 1024 ? 120 * 1024 : USED;
  static_assert(END <= 232448, "shared memory");
};

// NU: planes of the weighted keys; NS: planes of the state as an operand
template <int DK, int DV, int NU, int NS, bool OUT>
__global__ void __launch_bounds__(256, 1) tc_walk_kernel(const Walk p) {
  using Y = TLay<DK, DV, NU, NS, OUT>;
  constexpr int HV = DV / 2;                                   // value columns of a thread
  extern __shared__ __align__(1024) uint8_t sm[];
  Gates* gates = reinterpret_cast<Gates*>(sm + Y::G0);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, q4 = warp & 3, half = warp >> 2, row = 32 * q4 + lane;
  const int h = blockIdx.y;
  const Run run = find_run(p, blockIdx.x);
  if constexpr (OUT) {
    if (run.zlo < run.zhi)
      for (int64_t i = tid; i < (run.zhi - run.zlo) * p.vd; i += 256)
        st_any(p.out, !p.out_f32, ((run.zlo + i / p.vd) * p.H + h) * p.vd + i % p.vd, 0.f);
    if (p.count_bad && run.any && run.first && blockIdx.y == 0 && tid == 0) {
      const int64_t a = p.cu ? p.cu[run.s] : 0, b = p.cu ? p.cu[run.s + 1] : 0;
      if (p.cu && (a < 0 || b < a || b > p.T || (run.s == 0 && a != 0))) atomicAdd(&g_bad_offsets, 1u);
    }
  }
  if (!run.any) return;
  // the run that the sequence is left through has nobody to pass its sum to
  if (!OUT && (p.rev ? run.first : run.last)) return;

  const uint32_t base = smem_u32(sm), bar = base + Y::BAR;      // Q K^T, Q S, P V, U; tensor memory address
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(bar + 8 * i, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(bar + 32, 512);
    tmem_relinquish();
  }
  const int64_t sh = run.s * p.H + h, dd = (int64_t)p.kd * p.vd, slot_h = (int64_t)blockIdx.x * p.H + h;
  const int Hq = p.H / p.gq, Hk = p.H / p.gk, Hv = p.H / p.gv;
  const int len = (int)(run.hi - run.lo), chunks = (len + 127) / 128;
  const int64_t r0 = run.base + run.lo;                         // the run's first token
  const int64_t sk = (int64_t)Hk * p.kd, sv = (int64_t)Hv * p.vd, sq = (int64_t)Hq * p.kd;
  const bf16* gk = (const bf16*)p.k + r0 * sk + h / p.gk * p.kd;
  const bf16* gv = (const bf16*)p.v + r0 * sv + h / p.gv * p.vd;
  const bf16* gq = OUT ? (const bf16*)p.q + r0 * sq + h / p.gq * p.kd : nullptr;
  // chunk i of the walk; backwards in time (sums only) from the last one
  const auto first_of = [&](int i) { return 128 * (p.rev ? chunks - 1 - i : i); };
  const auto rows_of = [&](int i) { const int c0 = first_of(i); return len - c0 < 128 ? len - c0 : 128; };
  const auto kbuf = [&](int i) { return base + Y::K0 + (Y::NK == 2 ? (i & 1) * Y::TK : 0); };
  const auto load_q = [&](int i) { if (i < chunks) fetch128<DK>(base + Y::Q0, gq + first_of(i) * sq, sq, rows_of(i), p.kd); };
  const auto load_k = [&](int i) { if (i < chunks) fetch128<DK>(kbuf(i), gk + first_of(i) * sk, sk, rows_of(i), p.kd); };
  const auto load_v = [&](int i) { if (i < chunks) fetch128<DV>(base + Y::V0, gv + first_of(i) * sv, sv, rows_of(i), p.vd); };
  if constexpr (OUT) load_q(0);
  load_k(0);
  cp_commit();
  load_v(0);
  cp_commit();
  double total = 0.0;
  if (warp == 7 && chunks) total += scan_gates(gates_of(p, r0 + first_of(0), rows_of(0), h, lane), gates[0], lane);

  // the state: row `row` (a key feature), columns HV half + [0, HV)
  float S[HV];
  const int cols = row < p.kd ? p.vd - HV * half : 0;           // that there are of them
  if (!OUT) {
#pragma unroll
    for (int j = 0; j < HV; ++j) S[j] = 0.f;
  } else if (p.seg_state || p.init_f32) {
    const float* x = p.seg_state ? p.seg_state + slot_h * dd + row * p.sk + HV * half * p.sc : (const float*)p.init + sh * dd + row * p.ik + HV * half * p.ic;
    const int64_t d = p.seg_state ? p.sc : p.ic;
#pragma unroll
    for (int j = 0; j < HV; ++j, x += d) S[j] = j < cols ? *x : 0.f;
  } else {
    const bf16* x = (const bf16*)p.init + sh * dd + row * p.ik + HV * half * p.ic;
#pragma unroll
    for (int j = 0; j < HV; ++j, x += p.ic) S[j] = j < cols ? __bfloat162float(*x) : 0.f;
  }
  // its image for Q S: [feature][column], 64 columns a tile
  const auto put_state = [&]() {
    if (row < DK) {
#pragma unroll
      for (int j = 0; j < HV; j += 8) {
        uint32_t s[4][NS];
#pragma unroll
        for (int e = 0; e < 4; ++e) planes<NS>(S[j + 2 * e], S[j + 2 * e + 1], s[e]);
        const int c8 = (HV * half + j) / 8;
#pragma unroll
        for (int k = 0; k < NS; ++k)
          sts16(base + Y::S0 + k * Y::SP + (c8 >> 3) * DK * 128 + sw128_chunk(row, c8 & 7), make_uint4(s[0][k], s[1][k], s[2][k], s[3][k]));
      }
    }
  };
  if constexpr (OUT) put_state();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(bar + 32));
  const uint32_t tSC = tmem, tOI = tmem + 128, tOA = tmem + 256, tU = tmem + 384, lane_base = (uint32_t)(32 * q4) << 16;
  bool ok = true;
  const bool wide = p.vd % 16 == 0 && ((uintptr_t)p.out & 31) == 0;

  for (int i = 0; i < chunks; ++i) {
    const int nv = rows_of(i);
    const int64_t t0 = r0 + first_of(i);
    const uint32_t ph = i & 1, uk = kbuf(i), uv = base + Y::V0;
    const Gates& gs = gates[i & 1];
    if constexpr (OUT) {
      cp_wait<1>();                       // Q and K
      fence_async_smem();                 // (the state's image too)
      tc_fence_before();
      __syncthreads();
      if (tid == 0) {
        tc_fence_after();
        constexpr uint32_t d_qk = idesc_bf16(128, 128, 0, 0), d_qs = idesc_bf16(128, DV, 0, 1);
#pragma unroll
        for (int s = 0; s < DK / 16; ++s) umma_bf16(tSC, desc_kmajor(base + Y::Q0, 16384, s), desc_kmajor(uk, 16384, s), d_qk, s > 0);
        umma_commit(bar);
#pragma unroll
        for (int n = NS - 1; n >= 0; --n)
#pragma unroll
          for (int s = 0; s < DK / 16; ++s)
            umma_bf16(tOI, desc_kmajor(base + Y::Q0, 16384, s), desc_mnmajor(base + Y::S0 + n * Y::SP, DK * 128, s), d_qs, n < NS - 1 || s > 0);
        umma_commit(bar + 8);
      }
    }
    float4 gn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (warp == 7 && i + 1 < chunks) gn = gates_of(p, r0 + first_of(i + 1), rows_of(i + 1), h, lane);
    cp_wait<0>();                         // V (and, without Q, K)
    if constexpr (!OUT) __syncthreads();
    if constexpr (OUT) {
      if (ok) ok = mbar_wait(bar, ph);    // scores; K may be overwritten
      tc_fence_after();
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {
        const int grp = 2 * half + g;     // columns 32 grp + [0, 32)
        uint32_t pk[16];
        if (grp > q4) {
#pragma unroll
          for (int e = 0; e < 16; ++e) pk[e] = 0u;
        } else {
          uint32_t x[32];
          tmem_ld32(tSC + lane_base + 32 * grp, x);
          tmem_ld_wait();
          if (grp < q4) {
            const float rf = gs.rf[row];
            const float4* cf = reinterpret_cast<const float4*>(&gs.cf[q4 - 1][32 * grp]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float4 c = cf[e];
              pk[2 * e] = pack_bf16x2(__uint_as_float(x[4 * e]) * (rf * c.x), __uint_as_float(x[4 * e + 1]) * (rf * c.y));
              pk[2 * e + 1] = pack_bf16x2(__uint_as_float(x[4 * e + 2]) * (rf * c.z), __uint_as_float(x[4 * e + 3]) * (rf * c.w));
            }
          } else {
            const float2 li = gs.lam[row];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float4 l = *reinterpret_cast<const float4*>(&gs.lam[32 * grp + 2 * e]);
              const float a = 2 * e <= lane ? __uint_as_float(x[2 * e]) * decay_of(li, make_float2(l.x, l.y)) : 0.f;
              const float b = 2 * e + 1 <= lane ? __uint_as_float(x[2 * e + 1]) * decay_of(li, make_float2(l.z, l.w)) : 0.f;
              pk[e] = pack_bf16x2(a, b);
            }
          }
        }
        // P over its own half of SC: 64 half + [0, 32)
        tmem_st16(tSC + lane_base + 64 * half + 16 * g, pk);
      }
      tmem_st_wait();
    }
    weigh<DK, NU>(uk, base + Y::L0, Y::TK, gs.wt, p.rev);
    bool odd = false;
    if constexpr (OUT) odd = odd_values<DV>(uv);
    fence_async_smem();
    tc_fence_before();
    odd = __syncthreads_or(odd) != 0;
    if (tid == 0) {
      tc_fence_after();
      constexpr uint32_t d_pv = idesc_bf16(128, DV, 0, 1), d_u = idesc_bf16(128, DV, 1, 1);
      if constexpr (OUT) {
#pragma unroll
        for (int s = 0; s < 8; ++s) umma_ts(tOA, tSC + 64 * (s >> 2) + 8 * (s & 3), desc_mnmajor(uv, 16384, s), d_pv, s > 0);
        umma_commit(bar + 16);
      }
#pragma unroll
      for (int n = NU - 1; n >= 0; --n)
#pragma unroll
        for (int s = 0; s < 8; ++s)
          umma_bf16(tU, desc_mnmajor(n ? base + Y::L0 + (n - 1) * Y::TK : uk, 16384, s), desc_mnmajor(uv, 16384, s), d_u, n < NU - 1 || s > 0);
      umma_commit(bar + 24);
    }
    if (warp == 7 && i + 1 < chunks) total += scan_gates(gn, gates[(i + 1) & 1], lane);
    if constexpr (OUT) {
      if (ok) ok = mbar_wait(bar + 8, ph);          // Q S: Q may be overwritten
      load_q(i + 1);
      if constexpr (Y::NK == 2) load_k(i + 1);
      cp_commit();
      if (ok) ok = mbar_wait(bar + 16, ph);
      tc_fence_after();
      if (odd) masked_sums<DV, false>(tSC + lane_base, tOA + lane_base, uv, row, half);
      const float wi = gs.wt[row].x;
      const int64_t at = ((t0 + row) * p.H + h) * p.vd + HV * half;
      const int64_t ra = p.r ? ((t0 + row) * (p.H / p.gr) + h / p.gr) * p.vd + HV * half : 0;
      float dot = 0.f;
#pragma unroll 1
      for (int c0 = 0; c0 < HV; c0 += 16) {
        uint32_t a[16], b[16];
        tmem_ld16(tOI + lane_base + HV * half + c0, a);
        tmem_ld16(tOA + lane_base + HV * half + c0, b);
        tmem_ld_wait();
        if (row < nv) {
          if (p.r) {
            // the row's product with what comes from before the chunk
#pragma unroll
            for (int e = 0; e < 16; e += 8)
              if (HV * half + c0 + e < p.vd) {
                const uint4 u = __ldg((const uint4*)((const bf16*)p.r + ra + c0 + e));
                const uint32_t y[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float2 z = pair_of(y[k]);
                  dot = fmaf(__uint_as_float(a[e + 2 * k]), z.x, fmaf(__uint_as_float(a[e + 2 * k + 1]), z.y, dot));
                }
              }
          }
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = fmaf(wi, __uint_as_float(a[e]), __uint_as_float(b[e]));
          const int left = p.vd - (HV * half + c0);
          if (p.out_f32) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              if (e < left) *reinterpret_cast<float4*>((float*)p.out + at + c0 + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
            bf16* d = (bf16*)p.out + at + c0;
            if (wide) {
              if (left > 0) st_global_v8(d, w);
            } else {
              if (left > 0) *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
              if (left > 8) *reinterpret_cast<uint4*>(d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
        }
      }
      if (p.r && row < nv) p.rdot[(half * (p.cu ? p.T : p.nseq * p.T) + t0 + row) * p.H + h] = wi * dot;
    }
    if (ok) ok = mbar_wait(bar + 24, ph);           // U: K and V may be overwritten
    tc_fence_after();
    if constexpr (Y::NK == 1) load_k(i + 1);
    if constexpr (Y::NK == 1 && OUT) cp_commit();
    load_v(i + 1);
    cp_commit();
    const float all = gs.wt[127].x;
#pragma unroll
    for (int c0 = 0; c0 < HV; c0 += 16) {
      uint32_t u[16];
      tmem_ld16(tU + lane_base + HV * half + c0, u);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e) S[c0 + e] = fmaf(all, S[c0 + e], __uint_as_float(u[e]));
    }
    if constexpr (OUT) put_state();
  }
  if (!ok && lane == 0) atomicAdd(&g_wait_timeouts, 1u);
  cp_wait<0>();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);

  if constexpr (OUT) {
    if (run.last) {
      const int64_t at = sh * dd + row * p.ik + HV * half * p.ic;
      float* f = p.fin_f32 ? (float*)p.fin + at : p.fin32 + at;
      if (p.fin_f32 ? p.fin != nullptr : p.fin32 != nullptr)
#pragma unroll
        for (int j = 0; j < HV; ++j, f += p.ic)
          if (j < cols) *f = S[j];
      if (p.fin_f32 && p.fin32) {
        f = p.fin32 + at;
#pragma unroll
        for (int j = 0; j < HV; ++j, f += p.ic)
          if (j < cols) *f = S[j];
      }
      if (!p.fin_f32 && p.fin) {
        bf16* o = (bf16*)p.fin + at;
#pragma unroll
        for (int j = 0; j < HV; ++j, o += p.ic)
          if (j < cols) *o = __float2bfloat16_rn(S[j]);
      }
    }
  } else {
    if (warp == 7 && lane == 0) p.seg_total[slot_h] = total;
    float* f = p.seg_state + slot_h * dd + (int64_t)HV * half * p.kd + row;
#pragma unroll
    for (int j = 0; j < HV; ++j, f += p.kd)
      if (j < cols) *f = S[j];
  }
}

template <int DK, int DV, int NU, int NS, bool OUT>
int launch_tc(cudaStream_t stream, const Walk& p, const char* name) {
  using Y = TLay<DK, DV, NU, NS, OUT>;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(tc_walk_kernel<DK, DV, NU, NS, OUT>, Y::END));
  ProfScope ps(name, stream);
  tc_walk_kernel<DK, DV, NU, NS, OUT><<<dim3((unsigned)p.nslots, (unsigned)p.H), 256, Y::END, stream>>>(p);
  GLA_CHECK_LAUNCH();
  return GLA_OK;
}
unsigned int tc_walk_timeouts();

}  // namespace decay
}  // namespace gla
