// The walks of gla_decay.cuh on the fifth-generation tensor cores: bf16, head sizes up to 128, 128 tokens at a time.
//
// Per chunk:  SC = Q K^T,  OI = Q S,  OA = P V  and  U = (w K)^T V  (w = exp(lam_L - lam_j), in two or three bf16 planes).  Eight
// warps turn SC into P in tensor memory (a thread per row and half of the columns), weigh K in place, write exp(lam_i) OI + OA,
// and keep the state in registers: S <- exp(lam_L) S + U, from where its bf16 image goes to shared memory for the next chunk.
// One warp issues the products, one the tensor copies, one prepares the gates of the chunk to come.
//
// Why.  The same walk in mma.sync spends 14,000 instructions per 64 tokens, of which 1900 multiply: operand fragments, their
// conversion and the accumulators' addressing are the work.  Here operands go from shared memory to the tensor cores as the
// copies left them.
//
// What bounds it (4 x 4096 tokens of 6 heads, 128 x 128, runs of 768 tokens: 47 us a walk with outputs, 22 us one of sums).  A walk of
// n chunks takes 21 + 4.8 n us (144 blocks, n from 1 to 32, caches cold).  A chunk's 9000 cycles are its phases in a row, since
// each needs the one before: scores 1900, weights 1100, the check of the values 600, a wait for the products 1100, outputs and
// their stores 3000, the state 600.  No unit is at work for a third of them (tensor cores 19 %, accesses to shared memory 17 %, HBM
// 24 %), and there is room for one block per SM only.  The 21 us are what comes before the first chunk, the entering state read in
// strides among it, and after the last.  Measured besides: sixteen workers the same; eight for the scores and eight for outputs
// and state side by side 49 to 57 us.
//
// Roundings.  P and the state's image are one bf16 plane, as in this library's other chunk kernels: 2^-9 of each term, which leaves
// outputs 2.3e-3 of their norm off, where their own rounding to bf16 is 1.7e-3.  Two planes of the state cost its second product and
// the second stage of K: 8.2 us a chunk instead of 4.8, which only a backward with the gates' gradient is worth, whose terms cancel;
// there P has two planes as well (9.0 us a chunk).  The state itself, its sums and the gates' are in 32 bits and more.
//
// Tiles: 128 rows x 64 columns of bf16, 128-byte rows, 16-byte pieces at piece ^ (row % 8) (tc_ptx.cuh); D columns are D / 64
// of them.  A copy brings 128 rows whatever the sequence's length: rows past its end are another sequence's or beyond the
// array (zeros), and are zeroed where a product would meet them (keys as they are weighed, values in place).
#pragma once
#include "gla_decay.cuh"
#include "tma_maps.cuh"

namespace gla {
namespace decay {

using namespace tc;

__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
         "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
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

// `cols` (a multiple of 8, at most N) elements side by side, from or to an address that may be anything its type allows
template <int N>
__device__ __forceinline__ void load_side(float (&S)[N], const void* p, int f32, int cols) {
  const bool vec = ((uintptr_t)p & 15) == 0;
#pragma unroll
  for (int j = 0; j < N; j += 8) {
    float* s = S + j;
    if (j >= cols) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = 0.f;
    } else if (!vec) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = ld_any(p, !f32, j + e);
    } else if (f32) {
      const float4 a = *reinterpret_cast<const float4*>((const float*)p + j), b = *reinterpret_cast<const float4*>((const float*)p + j + 4);
      s[0] = a.x; s[1] = a.y; s[2] = a.z; s[3] = a.w; s[4] = b.x; s[5] = b.y; s[6] = b.z; s[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>((const bf16*)p + j);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) { const float2 y = pair_of(u[e]); s[2 * e] = y.x; s[2 * e + 1] = y.y; }
    }
  }
}
template <int N>
__device__ __forceinline__ void store_side(const float (&S)[N], void* p, int f32, int cols) {
  const bool vec = ((uintptr_t)p & 15) == 0;
#pragma unroll
  for (int j = 0; j < N; j += 8) {
    const float* s = S + j;
    if (j >= cols) continue;
    if (!vec) {
#pragma unroll
      for (int e = 0; e < 8; ++e) st_any(p, !f32, j + e, s[e]);
    } else if (f32) {
      *reinterpret_cast<float4*>((float*)p + j) = make_float4(s[0], s[1], s[2], s[3]);
      *reinterpret_cast<float4*>((float*)p + j + 4) = make_float4(s[4], s[5], s[6], s[7]);
    } else {
      *reinterpret_cast<uint4*>((bf16*)p + j) = make_uint4(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]), pack_bf16x2(s[4], s[5]), pack_bf16x2(s[6], s[7]));
    }
  }
}

static __device__ unsigned int g_wait_timeouts = 0;
static inline unsigned int read_wait_timeouts() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_wait_timeouts, sizeof(v));
  return v;
}

// Looks at three barriers at once (a look takes some 200 cycles, done or not).
__device__ __forceinline__ bool all_done(uint32_t a, uint32_t pa, uint32_t b, uint32_t pb, uint32_t c, uint32_t pc) {
  uint32_t x, y, z;
  asm volatile("{\n\t.reg .pred p, q, r;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%3], %4;\n\t"
               "mbarrier.test_wait.parity.shared::cta.b64 q, [%5], %6;\n\tmbarrier.test_wait.parity.shared::cta.b64 r, [%7], %8;\n\t"
               "selp.u32 %0, 1, 0, p;\n\tselp.u32 %1, 1, 0, q;\n\tselp.u32 %2, 1, 0, r;\n\t}\n"
               : "=r"(x), "=r"(y), "=r"(z) : "r"(a), "r"(pa), "r"(b), "r"(pb), "r"(c), "r"(pc) : "memory");
  return x && y && z;
}
// (tokens, heads, D) seen as 3-d (d, head, token); box 64 x 1 x 128, columns past D zeros
inline int make_map_tokens(CUtensorMap* m, const void* ptr, int64_t rows, int64_t heads, int64_t D) {
  if (rows > 0x7fffffffLL) return GLA_ERR_TOO_LARGE;
  const MapKey key{ptr, rows, heads, 17, (int)D, 0, 0};
  if (const CUtensorMap* hit = map_cache().find(key)) { *m = *hit; return GLA_OK; }
  EncodeTiledFn fn = encode_fn();
  if (!fn) return GLA_ERR_NO_DEVICE;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows}, strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)(heads * D) * 2};
  cuuint32_t box[3] = {64, 1, 128}, estr[3] = {1, 1, 1};
  const auto encode = [&]() {
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // a host thread that has not launched yet (autograd's, in a process's first backward): selecting its device binds it
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return GLA_ERR_NO_DEVICE;
    r = encode();
  }
  if (r != CUDA_SUCCESS) return GLA_ERR_LAUNCH;
  map_cache().put(key, *m);
  return GLA_OK;
}
// A wait that looks before it sleeps; bounded like mbar_wait, and after one that ran out nothing waits any more.
__device__ __forceinline__ void wait_for(bool& ok, uint32_t bar, uint32_t parity) {
  if (!ok) return;
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  if (!done) ok = mbar_wait(bar, parity);
}

// Worker warps (eight: with sixteen, whose threads have half the registers, what does not fit them goes through an L1 that shared
// memory leaves next to nothing of); warps for products, copies, gates.  The workers stand side by side in TC_COLS groups of 128
// threads, a thread per row, and TC_ROWS of 8 threads a row.
constexpr int TC_WORK = 8, TC_THREADS = (TC_WORK + 3) * 32, TC_COLS = TC_WORK / 4, TC_ROWS = TC_WORK * 4;

// What a chunk of 128 needs of its gates, made by one warp, four rows a lane.  lam: running sums, base 2, as two floats;
// wt: exp(lam_i), exp(lam_L - lam_i).  With a the last token before i's group of 32 rows, the weight exp(lam_i - lam_j) of a pair
// is rf_i cf_j, cf[g - 1]: exp(lam_a - lam_j) for the tokens before group g, cd: for those of the group itself, as long as
// the sums move by at most `span` <= 80 inside it; where a gate is sharper, the weights inside a group are formed pair by pair.
struct alignas(16) Gates {
  float2 lam[128], wt[128];
  float rf[128], cd[128], cf[3][128];
  float span[4];
  // exp(-lam_j) and exp(lam_i - lam_L), and the largest |lam|, |lam_L - lam| (base 2).  As long as these are below MILD a product
  // of scores needs one weight a column, and what is left of the weights multiplies a row of the result, which what comes from
  // the state shares: both add up in one accumulator.
  float dn[128], up[128];
  float low, reach;
};
constexpr float MILD = 64.f;           // of the 127 that float32 and bf16 exponents reach: scores and sums below 2^63 stay finite
__device__ __forceinline__ float4 gates_of(const Walk& p, int64_t t0, int nv, int h, int lane) {
  float g[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) g[i] = 4 * lane + i < nv ? p.g[(t0 + 4 * lane + i) * p.gt + h] : 0.f;
  return make_float4(g[0], g[1], g[2], g[3]);
}
// Sums of two floats each (46 bits and more): a gate of -200 must not cost the weights behind it their last places, and doubles
// take five times as long.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  const float s = a.x + b.x, t = s - a.x, e = ((a.x - (s - t)) + (b.x - t)) + (a.y + b.y), h = s + e;
  return make_float2(h, e - (h - s));
}
__device__ __forceinline__ float2 scan_gates(float4 g, Gates& s, int lane) {
  const float x[4] = {g.x, g.y, g.z, g.w};
  float2 v[4], sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // exp of less than -200 is 0 either way; -inf would leave inf - inf
    const float y = x[i] < -200.f ? -200.f : x[i], hi = y * 1.44269504f, lo = fmaf(y, 1.44269504f, -hi) + y * 1.92596299e-8f;
    sum = add2(sum, make_float2(hi, lo));
    v[i] = sum;
  }
  float2 inc = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const float2 y = make_float2(__shfl_up_sync(0xffffffffu, inc.x, d), __shfl_up_sync(0xffffffffu, inc.y, d));
    if (lane >= d) inc = add2(inc, y);
  }
  const auto of = [&](int l) { return make_float2(__shfl_sync(0xffffffffu, inc.x, l), __shfl_sync(0xffffffffu, inc.y, l)); };
  const float2 all = of(31), at[3] = {of(7), of(15), of(23)}, left = make_float2(__shfl_up_sync(0xffffffffu, inc.x, 1), __shfl_up_sync(0xffffffffu, inc.y, 1));
  const float2 before = lane ? left : make_float2(0.f, 0.f), own = lane < 8 ? make_float2(0.f, 0.f) : lane < 16 ? at[0] : lane < 24 ? at[1] : at[2];
  float span = 0.f, low = 0.f, reach = 0.f;
  const auto most = [](float a, float b) { return !(b <= a) ? b : a; };          // (what is not a number stays)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = add2(before, v[i]);
    const float d = (y.x - own.x) + (y.y - own.y);
    const int r = 4 * lane + i;
    const float l = y.x + y.y, u = (all.x - y.x) + (all.y - y.y);
    span = most(span, fabsf(d));
    low = most(low, fabsf(l));
    reach = most(reach, fabsf(u));
    s.dn[r] = ex2(-l);
    s.up[r] = ex2(-u);
    s.lam[r] = y;
    s.wt[r] = make_float2(ex2(l), ex2(u));
    s.rf[r] = ex2(d);
    s.cd[r] = ex2(-d);
#pragma unroll
    for (int m = 0; m < 3; ++m)
      if (lane < 8 * (m + 1)) s.cf[m][r] = ex2((at[m].x - y.x) + (at[m].y - y.y));
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    if (d < 8) span = most(span, __shfl_xor_sync(0xffffffffu, span, d));
    low = most(low, __shfl_xor_sync(0xffffffffu, low, d));
    reach = most(reach, __shfl_xor_sync(0xffffffffu, reach, d));
  }
  if (lane == 0) { s.low = low; s.reach = reach; }
  if (lane % 8 == 0) s.span[lane / 8] = span;
  return all;
}
__device__ __forceinline__ float decay_of(float2 i, float2 j) { return ex2((i.x - j.x) + (i.y - j.y)); }

// Rows of a tile times a weight per row, in NU planes: the first in place, the others at lo, lo + plane, ...  Rows from nv on are
// zeros.
template <int D, int NU>
__device__ __forceinline__ void weigh(uint32_t tile, uint32_t lo, uint32_t plane, const float2* wt, bool rev, int nv) {
  const int r0 = threadIdx.x / 8, c = threadIdx.x % 8;
  const float* w_ = &wt[r0].x + (rev ? 0 : 1);
  const uint32_t at0 = sw128_chunk(r0, c);
#pragma unroll 2
  for (int j = 0; j < 128 / TC_ROWS; ++j) {
    const float w = w_[2 * TC_ROWS * j];
    uint4 x[D / 64];
#pragma unroll
    for (int b = 0; b < D / 64; ++b) x[b] = lds16(tile + b * 16384 + j * TC_ROWS * 128 + at0);
    if (r0 + TC_ROWS * j >= nv)
#pragma unroll
      for (int b = 0; b < D / 64; ++b) x[b] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint32_t at = b * 16384 + j * TC_ROWS * 128 + at0;
      const uint32_t u[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
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
// Rows from nv on become zeros; returns whether what is left holds something that is not finite (of the thread's pieces).
template <int D>
__device__ __forceinline__ bool check_rows(uint32_t tile, int nv) {
  const int r0 = threadIdx.x / 8, c = threadIdx.x % 8;
  const uint32_t at0 = tile + sw128_chunk(r0, c);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 128 / TC_ROWS; ++j)
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint32_t at = at0 + b * 16384 + j * TC_ROWS * 128;
      if (r0 + TC_ROWS * j < nv) {
        const uint4 v = lds16(at);
        m = __vmaxu2(__vmaxu2(m, v.x & 0x7fff7fffu), __vmaxu2(v.y & 0x7fff7fffu, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
      } else {
        sts16(at, make_uint4(0u, 0u, 0u, 0u));
      }
    }
  return (m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u;
}
// What is not finite in OA = P V, by sums over the tokens up to the row's own: in the product, zeros of P meet what is not finite
// in V, and 0 x inf is not a number, where the recurrence has it at its own token and after only.
// P: this lane's row in tensor memory, 16 tokens in 8 columns, the second of two planes (NP) in the 8 behind; 16 columns of V at a time.
template <int NP>
__device__ __forceinline__ constexpr int score_at(int s) { return NP == 1 ? 32 * (s >> 1) + 8 * (s & 1) : 16 * s; }      // of tokens 16 s on
template <int NP>
__device__ __forceinline__ void load_scores(uint32_t a, float (&s)[16]) {
  uint32_t pk[8], pl[8];
  tmem_ld8(a, pk);
  if constexpr (NP == 2) tmem_ld8(a + 8, pl);
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 y = pair_of(pk[j]), z = NP == 2 ? pair_of(pl[j]) : make_float2(0.f, 0.f);
    s[2 * j] = y.x + z.x;
    s[2 * j + 1] = y.y + z.y;
  }
}
// scores 2 j and 2 j + 1 of 16, and all of them to their place, over what they were made of
template <int NP>
__device__ __forceinline__ void set_scores(uint32_t (&r)[8 * NP], int j, float x, float y) {
  uint32_t z[NP];
  planes<NP>(x, y, z);
#pragma unroll
  for (int n = 0; n < NP; ++n) r[8 * n + j] = z[n];
}
template <int NP>
__device__ __forceinline__ void store_scores(uint32_t a, const uint32_t (&r)[8 * NP]) {
  if constexpr (NP == 2) tmem_st16(a, r);
  else tmem_st8(a, r);
}
template <int DV, int NP>
__device__ __noinline__ void masked_sums(uint32_t tp, uint32_t to, uint32_t tv, int row, int qt) {
#pragma unroll 1
  for (int c0 = qt * (DV / TC_COLS); c0 < (qt + 1) * (DV / TC_COLS); c0 += 16) {
    float o[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = 0.f;
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
        if (t <= row)
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
  static constexpr int NK = !OUT || NU + NS <= 3 ? 2 : 1, NV = OUT ? 1 : 2, NL = OUT || NU > 2 ? 1 : 2;   // stages of K, V, the lower planes
  static constexpr int TK = DK * 256, TV = DV * 256, SP = DK * DV * 2;
  static constexpr int Q0 = 0, K0 = Q0 + (OUT ? TK : 0), V0 = K0 + NK * TK, L0 = V0 + NV * TV, S0 = L0 + NL * (NU - 1) * TK;
  static constexpr int STG = S0 + (OUT ? NS * SP : 0), G0 = STG + (OUT && DK == 64 ? 128 * DV * 2 : 0), BAR = G0 + 2 * (int)sizeof(Gates);
  // (64 features make rows 0 to 63 of a product of 128: the others are made of the 16 KB behind the keys' tile, whatever is there)
  // outputs are put together in the state's image once it has been used (64 features: its rows are too few, they have a tile of
  // their own)
  static constexpr int O0 = DK == 64 ? STG : S0;
  static constexpr int USED = BAR + 192 + (DK == 64 ? 16384 : 0);
  // one block per SM, whatever the sizes: each takes all of the tensor memory
  static constexpr int END = USED < 120 * 1024 ? 120 * 1024 : USED;
  static_assert(END <= 232448, "shared memory");
};
// barriers, 8 bytes each from BAR on
enum TcBar { B_Q = 0, B_K = 1, B_V = 3, B_QK = 5, B_QS = 6, B_PV = 7, B_U = 8, B_P = 10, B_S = 12, B_G = 13, B_GFREE = 15, B_COUNT = 17, B_TMEM = 17, B_ODD = 18 };

struct TcWalk {
  CUtensorMap q, k, v;
  Walk w;
};

// NU: planes of the weighted keys; NS: planes of the state as an operand and of the scores
template <int DK, int DV, int NU, int NS, bool OUT>
__global__ void __launch_bounds__(TC_THREADS, 1) tc_walk_kernel(const __grid_constant__ TcWalk a) {
  using Y = TLay<DK, DV, NU, NS, OUT>;
  constexpr int HV = DV / TC_COLS;                             // value columns of a worker
  const Walk& p = a.w;
  extern __shared__ __align__(1024) uint8_t sm[];
  Gates* gates = reinterpret_cast<Gates*>(sm + Y::G0);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int h = blockIdx.y;
  grid_dep_wait();
  grid_dep_launch();
  const Run run = find_run(p, blockIdx.x);
  if constexpr (OUT)
    if (run.zlo < run.zhi)
      for (int64_t i = tid; i < (run.zhi - run.zlo) * p.vd; i += TC_THREADS)
        st_any(p.out, !p.out_f32, ((run.zlo + i / p.vd) * p.H + h) * p.vd + i % p.vd, 0.f);
  if (!run.any) return;
  // the run that the sequence is left through has nobody to pass its sum to
  if (!OUT && (p.rev ? run.first : run.last)) return;

  const uint32_t base = smem_u32(sm), bars = base + Y::BAR;
  const auto bar = [&](int b) { return bars + 8 * b; };
  if (tid == 0) {
    for (int i = 0; i < B_COUNT; ++i) mbar_init(bar(i), i == B_P || i == B_P + 1 || i == B_S || i == B_GFREE || i == B_GFREE + 1 ? TC_WORK : 1);
    asm volatile("st.shared.v2.u32 [%0], {%1, %1};" ::"r"(bar(B_ODD)), "r"(0) : "memory");
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(bar(B_TMEM), 512);
    tmem_relinquish();
  }
  const int64_t sh = run.s * p.H + h, dd = (int64_t)p.kd * p.vd, slot_h = (int64_t)blockIdx.x * p.H + h;
  const int len = (int)(run.hi - run.lo), chunks = (len + 127) / 128;
  const int64_t r0 = run.base + run.lo;                         // the run's first token
  // chunk i of the walk; backwards in time (sums only) from the last one
  const auto first_of = [&](int i) { return 128 * (p.rev ? chunks - 1 - i : i); };
  const auto rows_of = [&](int i) { const int c0 = first_of(i); return len - c0 < 128 ? len - c0 : 128; };
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(bar(B_TMEM)));
  const uint32_t tSC = tmem, tOI = tmem + 128, tOA = tmem + 256, tU = tmem + 384;      // (sums only: U in two stages, 0 and 384)
  const auto ubuf = [&](int i) { return OUT || (i & 1) ? tU : tmem; };
  bool ok = true;
  // whether the workers found values that are not finite in chunk i, whose P and V they then read behind the product
  const auto was_odd = [&](int i) {
    uint32_t x;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(bar(B_ODD) + 4 * (i & 1)) : "memory");
    return x == (uint32_t)(i + 1);
  };

  if (warp == TC_WORK) {
    // ================= products =================
    if (lane == 0) {
      const uint64_t dQ = desc_kmajor(base + Y::Q0, 16384, 0), dK = desc_kmajor(base + Y::K0, 16384, 0);
      const uint64_t dKm = desc_mnmajor(base + Y::K0, 16384, 0), dV = desc_mnmajor(base + Y::V0, 16384, 0);
      const uint64_t dL = desc_mnmajor(base + Y::L0, 16384, 0), dS = desc_mnmajor(base + Y::S0, DK * 128, 0);
      constexpr uint32_t i_qk = idesc_bf16(128, 128, 0, 0), i_qs = idesc_bf16(128, DV, 0, 1), i_pv = idesc_bf16(128, DV, 0, 1),
                         i_u = idesc_bf16(128, DV, 1, 1);
      const auto kcol = [](int s) { return (uint32_t)((s >> 2) * 16384 + (s & 3) * 32); };     // 16 columns of a K-major operand
      for (int i = 0; i < chunks; ++i) {
        const uint32_t ph = i & 1, kst = Y::NK == 2 ? (i & 1) * Y::TK : 0, kph = Y::NK == 2 ? (i >> 1) & 1 : ph;
        const int kb = Y::NK == 2 ? i & 1 : 0, vb = Y::NV == 2 ? i & 1 : 0;
        if constexpr (OUT) {
          wait_for(ok, bar(B_Q), ph);
          wait_for(ok, bar(B_K + kb), kph);
          if (i >= 1 && was_odd(i - 1)) wait_for(ok, bar(B_S), ph);      // (P is read until the chunk before is done with)
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < DK / 16; ++s) umma_bf16(tSC, desc_advance(dQ, kcol(s)), desc_advance(dK, kst + kcol(s)), i_qk, s > 0);
          umma_commit(bar(B_QK));
          wait_for(ok, bar(B_S), ph);              // the state's image; OI, OA and U of the chunk before are read
          tc_fence_after();
#pragma unroll
          for (int n = NS - 1; n >= 0; --n)
#pragma unroll
            for (int s = 0; s < DK / 16; ++s)
              umma_bf16(tOI, desc_advance(dQ, kcol(s)), desc_advance(dS, n * Y::SP + s * 2048), i_qs, n < NS - 1 || s > 0);
          umma_commit(bar(B_QS));
        }
        wait_for(ok, bar(B_P + (i & 1)), (i >> 1) & 1);      // P, the weighted keys, the values checked
        if constexpr (!OUT) wait_for(ok, bar(B_V + vb), (i >> 1) & 1);
        tc_fence_after();
        const uint32_t vst = vb * Y::TV;
        if constexpr (OUT) {
          const bool one = gates[i & 1].low <= MILD && !p.r && !was_odd(i);         // (on top of Q S)
          const uint32_t to = one ? tOI : tOA;
#pragma unroll
          for (int n = NS - 1; n >= 0; --n)
#pragma unroll
            for (int s = 0; s < 8; ++s) umma_ts(to, tSC + score_at<NS>(s) + 8 * n, desc_advance(dV, s * 2048), i_pv, one || n < NS - 1 || s > 0);
          umma_commit(bar(B_PV));
        }
        const uint32_t lst = Y::NL == 2 ? (i & 1) * (NU - 1) * Y::TK : 0;
#pragma unroll
        for (int n = NU - 1; n >= 0; --n)
#pragma unroll
          for (int s = 0; s < 8; ++s)
            umma_bf16(ubuf(i), n ? desc_advance(dL, lst + (n - 1) * Y::TK + s * 2048) : desc_advance(dKm, kst + s * 2048),
                      desc_advance(dV, vst + s * 2048), i_u, n < NU - 1 || s > 0);
        umma_commit(bar(B_U + (OUT ? 0 : i & 1)));
      }
    }
    __syncwarp();
  } else if (warp == TC_WORK + 1) {
    // ================= tensor copies =================
    if (lane == 0) {
      const int hq = h / p.gq, hk = h / p.gk, hv = h / p.gv;
      for (int i = 0; i < chunks; ++i) {
        const int z = (int)(r0 + first_of(i)), kb = Y::NK == 2 ? i & 1 : 0, vb = Y::NV == 2 ? i & 1 : 0;
        if constexpr (OUT) {
          if (i >= 1) wait_for(ok, bar(B_QS), (i - 1) & 1);
          mbar_arrive_expect_tx(bar(B_Q), Y::TK);
          for (int b = 0; b < DK / 64; ++b) tma_load_3d(base + Y::Q0 + b * 16384, &a.q, 64 * b, hq, z, bar(B_Q));
        }
        if constexpr (OUT) {
          // (with two stages of K: the values of the chunk before waited for the product that used this one)
          if (i >= 1 && Y::NK == 1) wait_for(ok, bar(B_U), (i - 1) & 1);
        } else {
          if (i >= 2) wait_for(ok, bar(B_U + (i & 1)), ((i - 2) >> 1) & 1);
        }
        mbar_arrive_expect_tx(bar(B_K + kb), Y::TK);
        for (int b = 0; b < DK / 64; ++b) tma_load_3d(base + Y::K0 + kb * Y::TK + b * 16384, &a.k, 64 * b, hk, z, bar(B_K + kb));
        if constexpr (OUT)
          if (i >= 1) {
            if (Y::NK == 2) wait_for(ok, bar(B_U), (i - 1) & 1);
            if (was_odd(i - 1)) wait_for(ok, bar(B_S), i & 1);
          }
        mbar_arrive_expect_tx(bar(B_V + vb), Y::TV);
        for (int b = 0; b < DV / 64; ++b) tma_load_3d(base + Y::V0 + vb * Y::TV + b * 16384, &a.v, 64 * b, hv, z, bar(B_V + vb));
      }
    }
    __syncwarp();
  } else if (warp == TC_WORK + 2) {
    // ================= gates =================
    double total = 0.0, all[2] = {0.0, 0.0};
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
    if (chunks) g = gates_of(p, r0 + first_of(0), rows_of(0), h, lane);
    for (int i = 0; i < chunks; ++i) {
      if (i >= 2) wait_for(ok, bar(B_GFREE + (i & 1)), ((i - 2) >> 1) & 1);
      // (a decay that no token changes makes the same of every whole chunk)
      if (p.gt != 0 || i < 2 || rows_of(i) != rows_of(i - 2)) {
        const float2 x = scan_gates(g, gates[i & 1], lane);
        all[i & 1] = (double)x.x + (double)x.y;
      }
      total += all[i & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_G + (i & 1)));
      if (i + 1 < chunks) g = gates_of(p, r0 + first_of(i + 1), rows_of(i + 1), h, lane);
    }
    if (!OUT && lane == 0) p.seg_total[slot_h] = total;
  } else {
    // ================= workers =================
    const int q4 = warp & 3, qt = warp >> 2, row = 32 * q4 + lane;
    const uint32_t lane_base = (uint32_t)(32 * q4) << 16;
    // the state: row `row` (a key feature), columns HV qt + [0, HV)
    float S[HV];
    const int cols = row < p.kd ? p.vd - HV * qt : 0;           // that there are of them
    if (!OUT) {
#pragma unroll
      for (int j = 0; j < HV; ++j) S[j] = 0.f;
    } else {
      const int64_t sk = p.seg_state ? p.sk : p.ik, sc = p.seg_state ? p.sc : p.ic, at = (p.seg_state ? slot_h : sh) * dd + row * sk + HV * qt * sc;
      const int f32 = p.seg_state != nullptr || p.init_f32;
      const char* x = (const char*)(p.seg_state ? (const void*)p.seg_state : p.init) + at * (f32 ? 4 : 2);
      if (sc == 1) {
        load_side<HV>(S, x, f32, cols);
      } else {
#pragma unroll
        for (int j = 0; j < HV; ++j) S[j] = j < cols ? ld_any(x, !f32, j * sc) : 0.f;
      }
    }
    // its image for Q S: [feature][column], 64 columns a tile
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
      if (lane == 0) mbar_arrive(bar(B_S));
    };
    const auto take_u = [&](int i) {
      const float all = gates[i & 1].wt[127].x;
#pragma unroll
      for (int c0 = 0; c0 < HV; c0 += 16) {
        uint32_t u[16];
        tmem_ld16(ubuf(i) + lane_base + HV * qt + c0, u);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) S[c0 + e] = fmaf(all, S[c0 + e], __uint_as_float(u[e]));
      }
    };
    for (int i = 0; i < chunks; ++i) {
      const int nv = rows_of(i), kb = Y::NK == 2 ? i & 1 : 0, vb = Y::NV == 2 ? i & 1 : 0;
      const uint32_t ph = i & 1, kph = Y::NK == 2 ? (i >> 1) & 1 : ph;
      const uint32_t uk = base + Y::K0 + kb * Y::TK, uv = base + Y::V0 + vb * Y::TV;
      const Gates& gs = gates[i & 1];
      bool mild = false;
      if constexpr (OUT) {
        if (!all_done(bar(B_G + (i & 1)), (i >> 1) & 1, bar(B_QK), ph, bar(B_K + kb), kph)) {
          wait_for(ok, bar(B_G + (i & 1)), (i >> 1) & 1);
          wait_for(ok, bar(B_K + kb), kph);
          wait_for(ok, bar(B_QK), ph);
        }
        tc_fence_after();
        mild = gs.low <= MILD && !p.r;
#pragma unroll 1
        for (int sb = qt * (8 / TC_COLS); sb < (qt + 1) * (8 / TC_COLS); ++sb) {
          const int grp = sb >> 1;          // columns 16 sb + [0, 16), of the group of 32
          uint32_t s[8 * NS];
          if (grp > q4) {
#pragma unroll
            for (int e = 0; e < 8 * NS; ++e) s[e] = 0u;
          } else {
            uint32_t x[16];
            tmem_ld16(tSC + lane_base + 16 * sb, x);
            tmem_ld_wait();
            const bool own = grp == q4;
            const int last = own ? lane - 16 * (sb & 1) : 15;          // the row's last column
            if (mild || !own || gs.span[q4] <= 80.f) {
              const float rf = mild ? 1.f : gs.rf[row];
              const float4* cf = reinterpret_cast<const float4*>(mild ? &gs.dn[16 * sb] : own ? &gs.cd[16 * sb] : &gs.cf[q4 - 1][16 * sb]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 c = cf[e];
                const float y0 = 4 * e <= last ? __uint_as_float(x[4 * e]) * (rf * c.x) : 0.f;
                const float y1 = 4 * e + 1 <= last ? __uint_as_float(x[4 * e + 1]) * (rf * c.y) : 0.f;
                const float y2 = 4 * e + 2 <= last ? __uint_as_float(x[4 * e + 2]) * (rf * c.z) : 0.f;
                const float y3 = 4 * e + 3 <= last ? __uint_as_float(x[4 * e + 3]) * (rf * c.w) : 0.f;
                set_scores<NS>(s, 2 * e, y0, y1);
                set_scores<NS>(s, 2 * e + 1, y2, y3);
              }
            } else {
              const float2 li = gs.lam[row];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float4 l = *reinterpret_cast<const float4*>(&gs.lam[16 * sb + 2 * e]);
                const float x0 = 2 * e <= last ? __uint_as_float(x[2 * e]) * decay_of(li, make_float2(l.x, l.y)) : 0.f;
                const float x1 = 2 * e + 1 <= last ? __uint_as_float(x[2 * e + 1]) * decay_of(li, make_float2(l.z, l.w)) : 0.f;
                set_scores<NS>(s, e, x0, x1);
              }
            }
          }
          // P over this thread's own part of SC, which it has read up to here
          store_scores<NS>(tSC + lane_base + score_at<NS>(sb), s);
        }
        tmem_st_wait();
      }
      if constexpr (!OUT) {
        const uint32_t bu = i >= Y::NL ? bar(B_U + ((i - Y::NL) & 1)) : bar(B_K + kb), pu = i >= Y::NL ? ((i - Y::NL) >> 1) & 1 : kph;
        if (!all_done(bar(B_G + (i & 1)), (i >> 1) & 1, bar(B_K + kb), kph, bu, pu)) {
          wait_for(ok, bar(B_G + (i & 1)), (i >> 1) & 1);
          wait_for(ok, bar(B_K + kb), kph);
        }
      }
      if constexpr (!OUT)
        if (i >= Y::NL) wait_for(ok, bar(B_U + ((i - Y::NL) & 1)), ((i - Y::NL) >> 1) & 1);      // (the lower planes' stage)
      weigh<DK, NU>(uk, base + Y::L0 + (Y::NL == 2 ? (i & 1) * (NU - 1) * Y::TK : 0), Y::TK, gs.wt, p.rev, nv);
      if constexpr (OUT)
        if (i == 0) put_state();            // (here, so that the state is on its way during the first scores)
      if (OUT || nv < 128) {
        wait_for(ok, bar(B_V + vb), Y::NV == 2 ? (i >> 1) & 1 : ph);
        const bool odd = check_rows<DV>(uv, nv);
        if (OUT && odd) asm volatile("st.shared.u32 [%0], %1;" ::"r"(bar(B_ODD) + 4 * (i & 1)), "r"(i + 1) : "memory");
      }
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_P + (i & 1)));
      if constexpr (OUT) {
        const int64_t t0 = r0 + first_of(i);
        wait_for(ok, bar(B_PV), ph);             // (and Q S, which was issued before)
        tc_fence_after();
        const bool odd = was_odd(i), one = mild && !odd;
        if (odd) masked_sums<DV, NS>(tSC + lane_base, tOA + lane_base, uv, row, qt);
        const float wi = gs.wt[row].x, wp = mild ? wi : 1.f;
        const int64_t at = ((t0 + row) * p.H + h) * p.vd + HV * qt;      // (float32 outputs)
        const int64_t ra = p.r ? ((t0 + row) * (p.H / p.gr) + h / p.gr) * p.vd + HV * qt : 0;
        float dot = 0.f;
#pragma unroll 2
        for (int c0 = 0; c0 < HV; c0 += 16) {
          uint32_t x[16], y[16];
          tmem_ld16(tOI + lane_base + HV * qt + c0, x);
          if (one) {
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = 0u;
          } else {
            tmem_ld16(tOA + lane_base + HV * qt + c0, y);
          }
          tmem_ld_wait();
          if (row < nv) {
            if (p.r) {
              // the row's product with what comes from before the chunk
#pragma unroll
              for (int e = 0; e < 16; e += 8)
                if (HV * qt + c0 + e < p.vd) {
                  const uint4 u = __ldg((const uint4*)((const bf16*)p.r + ra + c0 + e));
                  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const float2 z = pair_of(w[k]);
                    dot = fmaf(__uint_as_float(x[e + 2 * k]), z.x, fmaf(__uint_as_float(x[e + 2 * k + 1]), z.y, dot));
                  }
                }
            }
            float o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = fmaf(wi, __uint_as_float(x[e]), wp * __uint_as_float(y[e]));
            const int left = p.vd - (HV * qt + c0);
            if (p.out_f32) {
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                if (e < left) *reinterpret_cast<float4*>((float*)p.out + at + c0 + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            } else {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
              const int c8 = (HV * qt + c0) / 8;
              const uint32_t d = base + Y::O0 + (c8 >> 3) * 16384;
              sts16(d + sw128_chunk(row, c8 & 7), make_uint4(w[0], w[1], w[2], w[3]));
              sts16(d + sw128_chunk(row, (c8 & 7) + 1), make_uint4(w[4], w[5], w[6], w[7]));
            }
          }
        }
        if (!p.out_f32) {
          // the warp's 32 rows of HV columns, whole rows of them side by side
          constexpr int LR = HV / 8, RI = 32 / LR;             // lanes a row, rows at once
          __syncwarp();
          const int c8 = HV / 8 * qt + lane % LR;
          const uint32_t d = base + Y::O0 + (c8 >> 3) * 16384;
          bf16* o = (bf16*)p.out + ((t0 + 32 * q4 + lane / LR) * p.H + h) * p.vd + 8 * c8;
#pragma unroll
          for (int j = 0; j < 32; j += RI) {
            const int r = 32 * q4 + j + lane / LR;
            if (r < nv && 8 * c8 < p.vd) *reinterpret_cast<uint4*>(o) = lds16(d + sw128_chunk(r, c8 & 7));
            o += (int64_t)RI * p.H * p.vd;
          }
          __syncwarp();
        }
        if (p.r && row < nv) p.rdot[(qt * (p.cu ? p.T : p.nseq * p.T) + t0 + row) * p.H + h] = wi * dot;
        wait_for(ok, bar(B_U), ph);
        tc_fence_after();
        take_u(i);
        if (i + 1 < chunks) put_state();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_GFREE + (i & 1)));
      } else {
        // the product of this chunk runs while the sums of the one before are taken
        if (i >= 1) {
          wait_for(ok, bar(B_U + ((i - 1) & 1)), ((i - 1) >> 1) & 1);
          tc_fence_after();
          take_u(i - 1);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_GFREE + ((i - 1) & 1)));
        }
      }
    }
    if (!OUT && chunks) {
      wait_for(ok, bar(B_U + ((chunks - 1) & 1)), ((chunks - 1) >> 1) & 1);
      tc_fence_after();
      take_u(chunks - 1);
    }
    if constexpr (OUT) {
      if (run.last) {
        // (only the forward's own walk leaves its state: columns side by side)
        const int64_t at = sh * dd + row * p.ik + HV * qt;
        if (p.fin) store_side<HV>(S, p.fin_f32 ? (void*)((float*)p.fin + at) : (void*)((bf16*)p.fin + at), p.fin_f32, cols);
        if (p.fin32) store_side<HV>(S, p.fin32 + at, 1, cols);
      }
    } else {
      float* f = p.seg_state + slot_h * dd + (int64_t)HV * qt * p.kd + row;
#pragma unroll
      for (int j = 0; j < HV; ++j, f += p.kd)
        if (j < cols) *f = S[j];
    }
  }
  if (!ok && lane == 0) atomicAdd(&g_wait_timeouts, 1u);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int DK, int DV, int NU, int NS, bool OUT>
int launch_tc(cudaStream_t stream, const Walk& p, const char* name) {
  using Y = TLay<DK, DV, NU, NS, OUT>;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(tc_walk_kernel<DK, DV, NU, NS, OUT>, Y::END));
  TcWalk a;
  a.w = p;
  const int64_t rows = p.cu ? p.T : p.nseq * p.T;
  GLA_TRY(make_map_tokens(&a.k, p.k, rows, p.H / p.gk, p.kd));
  GLA_TRY(make_map_tokens(&a.v, p.v, rows, p.H / p.gv, p.vd));
  if (OUT) GLA_TRY(make_map_tokens(&a.q, p.q, rows, p.H / p.gq, p.kd));
  else a.q = a.k;
  ProfScope ps(name, stream);
  GLA_LAUNCHED(launch_overlapped(tc_walk_kernel<DK, DV, NU, NS, OUT>, dim3((unsigned)p.nslots, (unsigned)p.H), dim3(TC_THREADS), Y::END, stream, a));
  return GLA_OK;
}

}  // namespace decay
}  // namespace gla
