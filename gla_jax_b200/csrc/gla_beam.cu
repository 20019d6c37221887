// Decoding over recurrent states: the single-token step of attention with one decay per head, steps and copies that follow a
// beam search's parents, and the selection of the next beams.
//
// What a beam carries in a recurrent model is its state, so that going on with a beam means having its state: rows of a
// state tensor are (request, beam), and parents (requests, beams) names for each beam of a request the beam it goes on from.
#include <math_constants.h>
#include "gla_common.cuh"
#include "gla_decay.cuh"

namespace gla {
namespace beam {

using decay::cp16;
using decay::cp_commit;
using decay::cp_wait;
using decay::sm32;

static __device__ unsigned int g_bad_parents = 0;

// parents[j] of a request of K beams, held inside [0, K); `count`: whether this thread reports one that was not
__device__ __forceinline__ int parent_of(const int* parents, int64_t n, int K, int j, bool count) {
  const int x = parents[n * K + j];
  if (count && (x < 0 || x >= K)) atomicAdd(&g_bad_parents, 1u);
  return x < 0 ? 0 : x >= K ? K - 1 : x;
}

// ---- single-token steps ----------------------------------------------------------------------------------------------------
// S <- f S + k (x) v and o = q S for a row (request or beam) and head, f one number (KEYED = false) or one per key feature.
// A block owns W value columns: W / 4 lanes of four columns, 128 / (W / 4) row lanes.  The state is read and written once,
// which is all that counts (8 Dk Dv bytes against a few hundred).
struct Step {
  float* S;
  const float* g;                 // (rows, H) or (rows, H, Dk)
  const void *v, *k, *q;          // (rows, H, Dv), (rows, Hk, Dk)
  void* out;
  const int* parents;             // (rows / K, K) or NULL (K = 1)
  int H, share, Dk, Dv, K, bf, out_bf;
};
constexpr int SNT = 128;

// One row per block, its loads all in flight before the first is used.  Measured, 32 requests x 16 heads, 128 x 128, bf16: 13.5 us
// with k and q read by every thread for itself -> 12.8 us through shared memory (the bytes at the copy rate: 10.3).
template <int W, int RPT>
__global__ void __launch_bounds__(SNT) step_kernel(const Step p) {
  constexpr int CL = W / 4, RL = SNT / CL;
  __shared__ float red[4][W];
  __shared__ float kq[2][RPT * RL];
  const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
  const int tiles = (p.Dv + W - 1) / W, col = blockIdx.x % tiles * W;      // of the block's columns, the first
  const int64_t row = blockIdx.x / tiles;                         // (request, head)
  const int64_t b = row / p.H, h = row % p.H, kv = (b * (p.H / p.share) + h / p.share) * p.Dk;
  const int c0 = col + 4 * cl;
  const bool on = c0 < p.Dv;
  float* Sp = p.S + (row * p.Dk + rl) * (int64_t)p.Dv + c0;
  grid_dep_wait();
  grid_dep_launch();
  float4 s[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i)
    if (on && rl + i * RL < p.Dk) s[i] = *reinterpret_cast<const float4*>(Sp + (int64_t)i * RL * p.Dv);
  for (int i = threadIdx.x; i < p.Dk; i += SNT) {
    kq[0][i] = ld_any(p.k, p.bf, kv + i);
    kq[1][i] = ld_any(p.q, p.bf, kv + i);
  }
  const float f = expf(p.g[row]);
  float4 vv = make_float4(0.f, 0.f, 0.f, 0.f), acc = vv;
  if (on) {
    const int64_t at = row * p.Dv + c0;
    vv = make_float4(ld_any(p.v, p.bf, at), ld_any(p.v, p.bf, at + 1), ld_any(p.v, p.bf, at + 2), ld_any(p.v, p.bf, at + 3));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rl + i * RL;
    if (!on || r >= p.Dk) continue;
    const float kr = kq[0][r], qr = kq[1][r];
    float4 n;
    n.x = fmaf(f, s[i].x, kr * vv.x); n.y = fmaf(f, s[i].y, kr * vv.y);
    n.z = fmaf(f, s[i].z, kr * vv.z); n.w = fmaf(f, s[i].w, kr * vv.w);
    *reinterpret_cast<float4*>(Sp + (int64_t)i * RL * p.Dv) = n;
    acc.x = fmaf(qr, n.x, acc.x); acc.y = fmaf(qr, n.y, acc.y); acc.z = fmaf(qr, n.z, acc.z); acc.w = fmaf(qr, n.w, acc.w);
  }
#pragma unroll
  for (int d = CL; d < 32; d <<= 1) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, d); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, d);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, d); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, d);
  }
  if (threadIdx.x % 32 < CL) *reinterpret_cast<float4*>(&red[threadIdx.x / 32][4 * cl]) = acc;
  __syncthreads();
  const int c = col + threadIdx.x;
  if (threadIdx.x < W && c < p.Dv)
    st_any(p.out, p.out_bf, row * p.Dv + c, (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]));
}

// All K beams of a request per block: every beam's old columns go into shared memory (a thread's own elements, which it
// alone reads again), then each beam is stepped from its parent's and written to its own place.  Nothing is read after it
// was overwritten, so the step needs no second set of states, and moving states costs no pass of its own: a beam that
// nobody goes on from is not even read.
template <int W, bool KEYED>
__global__ void __launch_bounds__(SNT) step_beams_kernel(const Step p) {
  constexpr int CL = W / 4, RL = SNT / CL;
  extern __shared__ __align__(16) uint8_t sm[];
  const int rpt = (p.Dk + RL - 1) / RL;
  float4* old = reinterpret_cast<float4*>(sm);                                        // [K][rpt][SNT]
  float* red = reinterpret_cast<float*>(sm + (size_t)p.K * rpt * SNT * 16);           // [K][4][W]
  float* kq = red + p.K * 4 * W;                                                      // [K][k, q][Dk]
  float* vf = kq + 2 * p.K * p.Dk;                                                    // [K][v (W), exp(g), parent, 2 spare]
  const int cl = threadIdx.x % CL, rl = threadIdx.x / CL, warp = threadIdx.x / 32;
  const int tiles = (p.Dv + W - 1) / W, col = blockIdx.x % tiles * W;
  const int64_t group = blockIdx.x / tiles, n = group / p.H, h = group % p.H;
  const int c0 = col + 4 * cl;
  const bool on = c0 < p.Dv;
  grid_dep_wait();
  grid_dep_launch();
  // beams that are somebody's parent: a lane looks at one
  const int lane = threadIdx.x % 32;
  const int par = lane < p.K ? parent_of(p.parents, n, p.K, lane, col == 0 && h == 0 && warp == 0) : 0;
  const unsigned int used = __reduce_or_sync(0xffffffffu, lane < p.K ? 1u << par : 0u);
  for (int j = 0; j < p.K; ++j) {
    if (!((used >> j) & 1u)) continue;
    const float* Sp = p.S + (((n * p.K + j) * p.H + h) * p.Dk + rl) * (int64_t)p.Dv + c0;
    for (int i = 0; i < rpt; ++i)
      if (on && rl + i * RL < p.Dk) cp16(sm32(old + (j * rpt + i) * SNT + threadIdx.x), Sp + (int64_t)i * RL * p.Dv, true);
  }
  cp_commit();
  for (int i = threadIdx.x; i < p.K * p.Dk; i += SNT) {
    const int j = i / p.Dk, r = i % p.Dk;
    const int64_t b = n * p.K + j, kv = (b * (p.H / p.share) + h / p.share) * p.Dk + r;
    kq[2 * j * p.Dk + r] = ld_any(p.k, p.bf, kv);
    kq[(2 * j + 1) * p.Dk + r] = ld_any(p.q, p.bf, kv);
  }
  for (int i = threadIdx.x; i < p.K * W; i += SNT) {
    const int j = i / W, c = col + i % W;
    vf[j * (W + 4) + i % W] = c < p.Dv ? ld_any(p.v, p.bf, ((n * p.K + j) * p.H + h) * p.Dv + c) : 0.f;
  }
  if (warp == 0 && lane < p.K) {
    vf[lane * (W + 4) + W] = KEYED ? 0.f : expf(p.g[(n * p.K + lane) * p.H + h]);
    vf[lane * (W + 4) + W + 1] = __int_as_float(par);
  }
  cp_wait<0>();
  __syncthreads();
  for (int j = 0; j < p.K; ++j) {
    const float* vj = vf + j * (W + 4);
    const int from = __float_as_int(vj[W + 1]);
    const int64_t row = (n * p.K + j) * p.H + h;
    float* Sp = p.S + (row * p.Dk + rl) * (int64_t)p.Dv + c0;
    const float f1 = vj[W];
    const float* kj = kq + 2 * j * p.Dk;
    const float4 vv = *reinterpret_cast<const float4*>(vj + 4 * cl);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < rpt; ++i) {
      const int r = rl + i * RL;
      if (!on || r >= p.Dk) continue;
      const float f = KEYED ? expf(p.g[row * p.Dk + r]) : f1;
      const float kr = kj[r], qr = kj[p.Dk + r];
      const float4 s = old[(from * rpt + i) * SNT + threadIdx.x];
      float4 x;
      x.x = fmaf(f, s.x, kr * vv.x); x.y = fmaf(f, s.y, kr * vv.y);
      x.z = fmaf(f, s.z, kr * vv.z); x.w = fmaf(f, s.w, kr * vv.w);
      *reinterpret_cast<float4*>(Sp + (int64_t)i * RL * p.Dv) = x;
      acc.x = fmaf(qr, x.x, acc.x); acc.y = fmaf(qr, x.y, acc.y); acc.z = fmaf(qr, x.z, acc.z); acc.w = fmaf(qr, x.w, acc.w);
    }
#pragma unroll
    for (int d = CL; d < 32; d <<= 1) {
      acc.x += __shfl_xor_sync(0xffffffffu, acc.x, d); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, d);
      acc.z += __shfl_xor_sync(0xffffffffu, acc.z, d); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, d);
    }
    if (threadIdx.x % 32 < CL) *reinterpret_cast<float4*>(red + (j * 4 + warp) * W + 4 * cl) = acc;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.K * W; i += SNT) {
    const int j = i / W, c = i % W;
    if (col + c >= p.Dv) continue;
    const float* x = red + j * 4 * W + c;
    st_any(p.out, p.out_bf, ((n * p.K + j) * p.H + h) * p.Dv + col + c, (x[0] + x[W]) + (x[2 * W] + x[3 * W]));
  }
}

template <int RPT>
static int launch_step(cudaStream_t st, const Step& p, int64_t rows) {
  ProfScope ps("decay_step_kernel", st);
  GLA_LAUNCHED(launch_overlapped(step_kernel<32, RPT>, dim3((unsigned)((p.Dv + 31) / 32 * rows)), dim3(SNT), 0, st, p));
  return GLA_OK;
}
template <int W, bool KEYED>
static int launch_beams(cudaStream_t st, const Step& p, int64_t groups) {
  constexpr int RL = SNT / (W / 4);
  const size_t smem = (size_t)p.K * ((p.Dk + RL - 1) / RL) * SNT * 16 + (size_t)p.K * (4 * W + 2 * p.Dk + W + 4) * 4;
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(step_beams_kernel<W, KEYED>, 200 << 10));      // (32 beams of 256 features: 194 KB)
  ProfScope ps("step_beams_kernel", st);
  GLA_LAUNCHED(launch_overlapped(step_beams_kernel<W, KEYED>, dim3((unsigned)((p.Dv + W - 1) / W * groups)), dim3(SNT), smem, st, p));
  return GLA_OK;
}
// Columns per block: as many as leave room for five or six blocks on an SM, so that one block's copies run beside another's steps
// (16 requests of 4 beams, 16 heads of 128 x 64: 17 us with 16 columns, 25 with 32 and three blocks); below 16 the rows of a block no
// longer fill 64 bytes.  Half the copy rate: 1.4 rounds of blocks, each of which loads, waits and then stores.
template <bool KEYED>
static int step_beams(cudaStream_t st, const Step& p, int64_t groups) {
  const int64_t col = (int64_t)p.K * (p.Dk + 31) / 32 * 32 * 4;      // bytes of a column
  if (col * 32 <= 32 << 10) return launch_beams<32, KEYED>(st, p, groups);
  if (col * 16 <= 96 << 10) return launch_beams<16, KEYED>(st, p, groups);
  return launch_beams<4, KEYED>(st, p, groups);
}

// ---- moving states -------------------------------------------------------------------------------------------------------
constexpr int RT = 64;                 // tensors per launch
struct Tensors {
  uint8_t* p[RT];
  int64_t bytes[RT];                   // of a row
  unsigned int start[RT + 1];          // first block of each tensor
  int n, K, count;                     // beams; whether this launch reports parents that are none
  const int* parents;
};
constexpr int MNT = 256;

// A thread owns one `unit` (16 bytes where the rows allow) of all K rows of a request: those that others go on from are
// read, then those that change are written.
template <typename T>
__global__ void __launch_bounds__(MNT) reorder_kernel(const Tensors t) {
  extern __shared__ __align__(16) uint8_t sm[];
  T* old = reinterpret_cast<T*>(sm);                                   // [K][MNT]
  int i = 0, j = t.n;                                                  // the tensor of this block
  while (j - i > 1) {
    const int m = (i + j) / 2;
    if (t.start[m] <= blockIdx.x) i = m; else j = m;
  }
  const int64_t units = t.bytes[i] / (int64_t)sizeof(T), per = (units + MNT - 1) / MNT;
  const int64_t blk = blockIdx.x - t.start[i], n = blk / per, u = blk % per * MNT + threadIdx.x;
  T* base = reinterpret_cast<T*>(t.p[i]) + n * t.K * units + u;
  const bool count = t.count && i == 0 && blk % per == 0 && threadIdx.x == 0;
  unsigned int taken = 0, moved = 0;
  for (int b = 0; b < t.K; ++b) {
    const int from = parent_of(t.parents, n, t.K, b, count);
    if (from != b) { moved |= 1u << b; taken |= 1u << from; }
  }
  if (!moved || u >= units) return;
  if constexpr (sizeof(T) == 16) {
    for (int b = 0; b < t.K; ++b)
      if ((taken >> b) & 1u) cp16(sm32(old + b * MNT + threadIdx.x), base + b * units, true);
    cp_commit();
    cp_wait<0>();
  } else {
    for (int b = 0; b < t.K; ++b)
      if ((taken >> b) & 1u) old[b * MNT + threadIdx.x] = base[b * units];
  }
  for (int b = 0; b < t.K; ++b)
    if ((moved >> b) & 1u) base[b * units] = old[parent_of(t.parents, n, t.K, b, false) * MNT + threadIdx.x];
}
template <typename T>
static int launch_reorder(cudaStream_t st, const Tensors& t) {
  static SmemAttrOnce attr;
  GLA_TRY(attr.ensure(reorder_kernel<T>, 32 * MNT * sizeof(T)));
  ProfScope ps("reorder_kernel", st);
  reorder_kernel<T><<<t.start[t.n], MNT, (size_t)t.K * MNT * sizeof(T), st>>>(t);
  GLA_CHECK_LAUNCH();
  return GLA_OK;
}

// ---- selection -------------------------------------------------------------------------------------------------------------
// For each request the M best of its K V continuations by score[k] + log_softmax(logits[k])[v], the largest first, the
// lowest (beam, token) first among equal ones.
//
// Within a row the totals never fall as the logits rise, so that nothing but M candidates per part and its (maximum, sum) leaves the
// pass; a second kernel forms the totals of the candidates in 64 bits and orders them.  Totals of unequal logits can be equal (a
// score like -1e18 leaves none of a logit's digits), and among those it is the lowest place that counts, not the larger logit:
// where the last candidate of a part meets the M-th total, and a logit next to its own would too, that row is read again.
//
// A block streams a part of a row, its threads keep the running maximum and sum of exponentials of
// the softmax and their two largest logits, as values: a minimum and two maxima a logit, of which the larger is the running
// maximum as well; the tile that they came in is kept, and looked through at the end for where.
// The M-th largest of the threads' largest is a bound: M logits reach it.  Threads whose second reaches it too may have
// more, which is one in a part on average and is looked up again; where few threads hold most of the large logits (nothing
// that a model leaves, but a sorted row may), the M largest are found one after the other.
// Measured, 64 x 8 rows of 128000 bf16 logits, M = 16, the pass alone: lists in shared memory that are cut as they grow 136 us,
// a sorted list per warp 312 us, the two largest with their places 79 us, this 57 us (the bytes at the copy rate: 17.5); both
// kernels 70 us.  What bounds it: 64 registers leave room for four blocks on an SM, so that the 900 or so that have a live row come in
// two rounds of 592, the second half empty (40 % of the warps there could be, instructions in 57 % of the cycles, HBM at 24 %), with
// one tile of a part on its way.
// A key is (order of the value, lowest index first), 0: none.
typedef unsigned long long u64;
__device__ __forceinline__ unsigned int order_of(float x) {
  const unsigned int u = __float_as_uint(x + 0.f);                      // -0 is 0
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned int o) { return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ u64 key_of(float x, unsigned int i) { return ((u64)order_of(x) << 32) | (unsigned int)~i; }
constexpr float FMOST = 3.402823466e38f;
// what a logit counts as: not-a-number as one that is masked, +inf as the largest finite number
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -CUDART_INF_F), FMOST); }

__device__ __forceinline__ u64 warp_sorted(u64 x, int lane) {           // descending over the lanes
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const u64 y = __shfl_xor_sync(0xffffffffu, x, j);
      const bool keep_max = ((lane & j) == 0) == ((lane & k) == 0);
      x = keep_max ? (x > y ? x : y) : (x > y ? y : x);
    }
  return x;
}

constexpr int QNT = 256, QV = 16, TILE = QNT * QV;                      // threads, logits per thread and tile
constexpr int CAP = 1024;                                               // candidates of a part before the last cut
struct Select {
  const void* logits;
  const float* scores;
  const unsigned char* finished;
  int64_t V;
  int K, M, bf, parts;
  int64_t part;                     // logits of a part, a multiple of TILE
  int64_t pad;
  u64* cand;                        // [row][part][M]
  double2* sums;                    // [row][part]: maximum, sum of exponentials
  float* out_scores;
  long long* tokens;
  int* parents;
};

// exp(x - m) with x <= m: the difference first, which is exact where it counts
__device__ __forceinline__ float exp_of(float d) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d * 1.4426950408889634f));
  return y;
}

template <bool BF>
__global__ void __launch_bounds__(QNT) select_parts_kernel(const Select p) {
  __shared__ u64 list[CAP], tau_;
  __shared__ int cnt, more, who[QNT];
  __shared__ u64 below[QNT];
  __shared__ float wm[8];
  __shared__ double ws[8];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t row = blockIdx.x / p.parts, V = p.V;
  const int own_part = blockIdx.x % p.parts;
  grid_dep_wait();
  grid_dep_launch();
  u64* cand = p.cand + (row * p.parts + own_part) * p.M;
  const float score = p.scores[row];
  const bool dead = !(score > -CUDART_INF_F), done = p.finished && p.finished[row];
  if (dead || done) {
    // a beam that has ended has one continuation, one without a score has none: the others rank by their number alone
    if (tid < p.M) {
      u64 x = 0;
      if (own_part == 0) {
        const bool one = done && !dead;
        const int64_t i = !one ? tid : tid == 0 ? p.pad : tid - 1 < p.pad ? tid - 1 : tid;
        if (i < V) x = key_of(one && tid == 0 ? 0.f : -CUDART_INF_F, (unsigned int)i);
      }
      cand[tid] = x;
    }
    if (tid == 0) p.sums[row * p.parts + own_part] = own_part == 0 ? make_double2(0.0, 1.0) : make_double2(-CUDART_INF, 0.0);
    return;
  }
  // A thread's logits are the same whatever a row's address, so that equal rows have equal sums to the last bit and their
  // totals tie.  Rows that do not start on 16 bytes are put together from two aligned accesses.
  constexpr int E = BF ? 8 : 4, NV = QV / E, ES = BF ? 2 : 4;         // logits per 16 bytes, accesses per tile
  const char* base = (const char*)p.logits + row * V * ES;
  const auto w_of = [](int i) { return i / E; };                      // the access that logit i of a thread's tile came by
  const int shift = (int)((uintptr_t)base & 15) / ES;
  const int64_t lo = own_part * p.part, hi = lo + p.part < V ? lo + p.part : V;
  float s = 0.f;
  float v1 = -CUDART_INF_F, v2 = -CUDART_INF_F;      // the two largest (v1 is the running maximum), and the tiles that they came in
  int64_t t1 = lo, t2 = lo;
  uint4 raw[2 * NV];                  // the next tile's 16 bytes, and the 16 behind them where a row starts anywhere
  const auto whole = [&](int64_t e) { return shift ? e >= shift && e - shift + 2 * E <= V : e + E <= V; };
  const auto request = [&](int64_t t0) {
#pragma unroll
    for (int w = 0; w < NV; ++w) {
      const int64_t e = t0 + (int64_t)(w * QNT + tid) * E;
      if (t0 < hi && whole(e)) {
        raw[w] = __ldg((const uint4*)(base + (e - shift) * ES));
        if (shift) raw[NV + w] = __ldg((const uint4*)(base + (e - shift + E) * ES));
      }
    }
  };
  request(lo);
  for (int64_t t0 = lo; t0 < hi; t0 += TILE) {
    float x[QV];                      // (-inf where there is none)
#pragma unroll
    for (int w = 0; w < NV; ++w) {
      const int64_t e = t0 + (int64_t)(w * QNT + tid) * E;
      if (whole(e)) {
        uint4 u = raw[w];
        if (shift) {
          const uint4 n = raw[NV + w];
          const unsigned int z[8] = {u.x, u.y, u.z, u.w, n.x, n.y, n.z, n.w};
          unsigned int y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // 32 bits from byte 4 i + shift ES on: words by a chain of selects, bytes by a funnel shift
            unsigned int a = z[i], b = z[i + 1];
#pragma unroll
            for (int j = 1; j < 4; ++j)
              if (shift * ES / 4 == j) { a = z[i + j]; b = z[i + j + 1 < 8 ? i + j + 1 : 7]; }
            y[i] = __funnelshift_r(a, b, shift * ES % 4 * 8);
          }
          u = make_uint4(y[0], y[1], y[2], y[3]);
        }
        const unsigned int y[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (BF) { x[w * E + 2 * i] = __uint_as_float(y[i] << 16); x[w * E + 2 * i + 1] = __uint_as_float(y[i] & 0xffff0000u); }
          else x[w * E + i] = __uint_as_float(y[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          x[w * E + i] = -CUDART_INF_F;
          if (e + i < hi) x[w * E + i] = BF ? __bfloat162float(((const bf16*)base)[e + i]) : ((const float*)base)[e + i];
        }
      }
    }
    request(t0 + TILE);
    const float o1 = v1, o2 = v2;
    float t;
    const auto take = [&]() {
#pragma unroll
      for (int i = 0; i < QV; ++i) {
        v2 = fmaxf(v2, fminf(v1, x[i]));
        v1 = fmaxf(v1, x[i]);
      }
      t = 0.f;
      if (v1 > -CUDART_INF_F) {
#pragma unroll
        for (int i = 0; i < QV; ++i) t += exp_of(x[i] - v1);
      }
    };
    take();
    if (t != t) {                      // +inf or what is not a number is among them
#pragma unroll
      for (int i = 0; i < QV; ++i) x[i] = clean(x[i]);
      v1 = o1;
      v2 = o2;
      take();
    }
    if (v1 > o1) {
      s *= exp_of(o1 - v1);
      if (v2 == o1) t2 = t1;           // (the first before is the second now, also among equal ones)
      else t2 = t0;
      t1 = t0;
    } else if (v2 > o2) {
      t2 = t0;
    }
    s += t;
  }
  const auto logit = [&](int64_t e) { return clean(BF ? __bfloat162float(((const bf16*)base)[e]) : ((const float*)base)[e]); };
  // the first of a tile's logits that is v, other than `but` (-1: none)
  const auto find = [&](int64_t t0, float v, int but) {
    int at = -1;
#pragma unroll
    for (int i = QV - 1; i >= 0; --i) {
      const int64_t e = t0 + (w_of(i) * QNT + tid) * E + i % E;
      if (e < hi && e != but && logit(e) == v) at = (int)e;
    }
    return at;
  };
  const int i1 = find(t1, v1, -1), i2 = find(t2, v2, i1);
  const float m = v1;
  // the bound: sorted by warp, a key's place among all is its place in its warp and what is larger in the others
  const u64 first = i1 < 0 ? 0 : key_of(v1, (unsigned int)i1), second = i2 < 0 ? 0 : key_of(v2, (unsigned int)i2);
  const u64 own = warp_sorted(first, lane);
  below[tid] = own;
  if (tid == 0) { tau_ = 1; cnt = 0; more = 0; }
  __syncthreads();
  {
    int place = lane;
    for (int w = 0; w < 8; ++w) {
      if (w == warp) continue;
      const u64* l = below + 32 * w;
      int n = 0;                       // of the 32, in descending order, those above
#pragma unroll
      for (int d = 16; d; d >>= 1)
        if (l[n + d - 1] > own) n += d;
      place += n + (n == 31 && l[31] > own);
    }
    if (own && place == p.M - 1) tau_ = own;
  }
  __syncthreads();
  const u64 tau = tau_;
  // (the table is read by now)
  if (first >= tau) list[atomicAdd(&cnt, 1)] = first;
  if (second >= tau) {
    list[atomicAdd(&cnt, 1)] = second;
    const int i = atomicAdd(&more, 1);
    who[i] = tid;
    below[i] = second;
  }
  __syncthreads();
  const int tiles = hi > lo ? (int)((hi - lo + TILE - 1) / TILE) : 0;
  for (int k = 0; k < more; ++k) {
    // the logits that thread who[k] met, below its second
    for (int j = tid; j < tiles * QV; j += QNT) {
      const int64_t e = lo + (int64_t)(j / QV) * TILE + (w_of(j % QV) * QNT + who[k]) * E + j % QV % E;
      if (e < V) {
        const u64 y = key_of(logit(e), (unsigned int)e);
        if (y >= tau && y < below[k]) {
          const int at = atomicAdd(&cnt, 1);
          if (at < CAP) list[at] = y;
        }
      }
    }
  }
  __syncthreads();
  const int n = cnt;
  if (n <= CAP) {
    for (int i = tid; i < n; i += QNT) {
      const u64 y = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[j] > y;
      if (rank < p.M) cand[rank] = y;
    }
    if (tid >= n && tid < p.M) cand[tid] = 0;
  } else {
    u64 prev = ~0ull;
    for (int k = 0; k < p.M; ++k) {
      u64 y = 0;
      for (int64_t e = lo + tid; e < hi; e += QNT) {
        const u64 z = key_of(logit(e), (unsigned int)e);
        if (z < prev && z > y) y = z;
      }
      y = warp_sorted(y, lane);
      if (lane == 0) below[warp] = y;
      __syncthreads();
      y = below[0];
      for (int w = 1; w < 8; ++w) y = below[w] > y ? below[w] : y;
      prev = y;
      if (tid == 0) cand[k] = y;
      __syncthreads();
    }
  }
  // (maximum, sum) of the part
  float top = m;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) wm[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, wm[w]);
  double sum = m > -CUDART_INF_F ? (double)s * exp_of(m - top) : 0.0;
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) ws[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
    for (int w = 0; w < 8; ++w) sum += ws[w];
    p.sums[row * p.parts + own_part] = make_double2(top, sum);
  }
}

// order of a 64-bit total, and the totals' candidates: (total, beam and token)
__device__ __forceinline__ u64 order_of(double x) {
  const long long u = __double_as_longlong(x + 0.0);
  return u < 0 ? ~(u64)u : (u64)u | 0x8000000000000000ull;
}
constexpr int SCAP = 1024, BNT = 512;   // candidates of a request: K parts M, at most; threads
__global__ void __launch_bounds__(BNT) select_beams_kernel(const Select p) {
  __shared__ u64 key[SCAP], where[SCAP];  // total's order; (beam, token)
  __shared__ double base[32][2];          // per beam: maximum, log of the sum
  __shared__ u64 cut_;                    // the M-th total
  __shared__ unsigned int doubt_;         // beams to be read again
  __shared__ int above, hits[BNT / 32];
  const int tid = threadIdx.x, K = p.K, M = p.M, per = p.parts * M, n = K * per;
  const int64_t req = blockIdx.x;
  grid_dep_wait();
  if (tid == 0) { doubt_ = 0; above = 0; }
  for (int k = tid / 32; k < K; k += BNT / 32) {
    const double2* sm = p.sums + (req * K + k) * p.parts;
    double top = -CUDART_INF, s = 0.0;
    for (int i = tid % 32; i < p.parts; i += 32) top = fmax(top, sm[i].x);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, d));
    for (int i = tid % 32; i < p.parts; i += 32)
      if (sm[i].x > -CUDART_INF) s += sm[i].y * exp(sm[i].x - top);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (tid % 32 == 0) { base[k][0] = top; base[k][1] = log(s); }
  }
  __syncthreads();
  const u64* cand = p.cand + req * n;
  const auto total = [&](int k, float x) {
    double t = -CUDART_INF;
    if (x > -CUDART_INF_F && base[k][0] > -CUDART_INF) t = (double)p.scores[req * K + k] + (((double)x - base[k][0]) - base[k][1]);
    if (!(t > -CUDART_INF)) t = -CUDART_INF;
    return order_of(t);
  };
  for (int i = tid; i < n; i += BNT) {
    const u64 c = cand[i];
    const int k = i / per;
    key[i] = c ? total(k, value_of((unsigned int)(c >> 32))) : 0;
    where[i] = ((u64)k << 32) | (unsigned int)~(unsigned int)c;
  }
  __syncthreads();
  // a candidate's place is the number of larger ones, counted by eight lanes
  const int part = tid % 8;
  for (int i0 = 0; i0 < n; i0 += BNT / 8) {
    const int i = i0 + tid / 8;
    const u64 x = i < n ? key[i] : 0, at = i < n ? where[i] : 0;
    int rank = 0;
    if (x)
#pragma unroll 4
      for (int j = part; j < n; j += 8) rank += key[j] > x || (key[j] == x && where[j] < at);
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, d);
    if (x && part == 0 && rank < M) {
      const long long u = (x >> 63) ? (long long)(x & 0x7fffffffffffffffull) : (long long)~x;
      p.out_scores[req * M + rank] = (float)__longlong_as_double(u);
      p.tokens[req * M + rank] = (long long)(at & 0xffffffffu);
      p.parents[req * M + rank] = (int)(at >> 32);
      if (rank == M - 1) cut_ = x;
    }
  }
  __syncthreads();
  const u64 cut = cut_;
  for (int i = tid; i < K * p.parts; i += BNT) {
    const int k = i / p.parts, last = i * M + M - 1;
    // (a beam that has ended or has no score left its tokens in order)
    if (key[last] != cut || !(p.scores[req * K + k] > -CUDART_INF_F) || (p.finished && p.finished[req * K + k]) || !(base[k][0] > -CUDART_INF)) continue;
    const unsigned int o = (unsigned int)(cand[last] >> 32), step = p.bf ? 0x10000u : 1u;
    const float x = value_of(o), up = clean(value_of(o + step));
    float down = value_of(o - step);
    if (down == x) down = value_of(o - 2 * step);                       // (-0)
    if (x > -CUDART_INF_F && ((up != x && total(k, up) == cut) || total(k, down) == cut)) atomicOr(&doubt_, 1u << k);
  }
  __syncthreads();
  const unsigned int doubt = doubt_;
  if (!doubt) return;
  for (int i = tid; i < n; i += BNT) if (key[i] > cut) atomicAdd(&above, 1);
  __syncthreads();
  // the first of those that are equal to the M-th, by beam and token: from the logits where in doubt, else from the candidates
  const int warp = tid / 32;
  int at = above;
  for (int k = 0; k < K && at < M; ++k) {
    const bool again = (doubt >> k) & 1u;
    const int64_t row = (req * K + k) * p.V, len = again ? p.V : per;
    for (int64_t e0 = 0; e0 < len && at < M; e0 += BNT) {
      const int64_t e = e0 + tid;
      bool hit = false;
      if (e < len)
        hit = (again ? total(k, clean(p.bf ? __bfloat162float(((const bf16*)p.logits)[row + e]) : ((const float*)p.logits)[row + e])) : key[k * per + e]) == cut;
      const unsigned int mask = __ballot_sync(0xffffffffu, hit);
      if (tid % 32 == 0) hits[warp] = __popc(mask);
      __syncthreads();
      int place = at + __popc(mask & ((1u << tid % 32) - 1u));
      for (int w = 0; w < BNT / 32; ++w) {
        if (w < warp) place += hits[w];
        at += hits[w];
      }
      if (hit && place < M) {
        p.tokens[req * M + place] = again ? (long long)e : (long long)(where[k * per + e] & 0xffffffffu);
        p.parents[req * M + place] = k;
      }
      __syncthreads();
    }
  }
}

// Parts of a row: six blocks for each SM (four are resident, three in float32), few enough that a request's candidates fit.
static void plan(int64_t rows, int64_t V, int K, int M, int* parts, int64_t* part) {
  const int64_t tiles = (V + TILE - 1) / TILE;
  int64_t n = (6 * 148 + rows - 1) / rows;
  if (n > tiles) n = tiles;
  if (n > SCAP / (K * M)) n = SCAP / (K * M);
  if (n < 1) n = 1;
  *part = (tiles + n - 1) / n * TILE;
  *parts = (int)((V + *part - 1) / *part);
}

}  // namespace beam
unsigned int beam_bad_parents() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, beam::g_bad_parents, sizeof(v));
  return v;
}
}  // namespace gla

using namespace gla;

extern "C" {

unsigned int gla_device_bad_parents(void) { return beam_bad_parents(); }

constexpr int64_t GRID_MOST = 2147483647;

static int step_check(int64_t B, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, int out_dtype, const int32_t* parents, int64_t K) {
  if (B <= 0 || H <= 0 || Hk <= 0 || Dk <= 0 || Dv <= 0 || H % Hk) return GLA_ERR_BAD_DIMS;
  if (parents && (K <= 0 || B % K)) return GLA_ERR_BAD_DIMS;
  if ((dtype != GLA_F32 && dtype != GLA_BF16) || (out_dtype != GLA_F32 && out_dtype != GLA_BF16)) return GLA_ERR_UNSUPPORTED;
  if (Dk % 8 || Dv % 8 || Dk > 256 || Dv > 256 || (parents && K > 32)) return GLA_ERR_UNSUPPORTED;
  if (B > GRID_MOST || B / (parents ? K : 1) * H > GRID_MOST / 64) return GLA_ERR_TOO_LARGE;      // (64 blocks of columns at most)
  return GLA_OK;
}

int gla_decay_step(void* stream, int64_t B, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, float* state, const float* log_decay,
                   const void* value, const void* key, const void* query, void* out, int out_dtype, const int32_t* parents, int64_t beams) {
  if (!state || !log_decay || !value || !key || !query || !out) return GLA_ERR_NULL_POINTER;
  GLA_TRY(step_check(B, H, Hk, Dk, Dv, dtype, out_dtype, parents, beams));
  if (!aligned16(state)) return GLA_ERR_ALIGNMENT;
  beam::Step p{state, log_decay, value, key, query, out, parents, (int)H, (int)(H / Hk), (int)Dk, (int)Dv, parents ? (int)beams : 1,
               dtype == GLA_BF16, out_dtype == GLA_BF16};
  cudaStream_t st = (cudaStream_t)stream;
  if (parents) return beam::step_beams<false>(st, p, B / beams * H);
  if (Dk <= 64) return beam::launch_step<4>(st, p, B * H);
  if (Dk <= 128) return beam::launch_step<8>(st, p, B * H);
  return beam::launch_step<16>(st, p, B * H);
}

int gla_decode_step_beams(void* stream, int64_t B, int64_t H, int64_t D, int dtype, float* state, const float* log_fgate, const void* value,
                          const void* key, const void* query, void* out, int out_dtype, const int32_t* parents, int64_t beams) {
  if (!state || !log_fgate || !value || !key || !query || !out || !parents) return GLA_ERR_NULL_POINTER;
  GLA_TRY(step_check(B, H, H, D, D, dtype, out_dtype, parents, beams));
  if (D != 32 && D != 64 && D != 128 && D != 256) return GLA_ERR_UNSUPPORTED;
  if (!aligned16(state)) return GLA_ERR_ALIGNMENT;
  beam::Step p{state, log_fgate, value, key, query, out, parents, (int)H, 1, (int)D, (int)D, (int)beams, dtype == GLA_BF16, out_dtype == GLA_BF16};
  return beam::step_beams<true>((cudaStream_t)stream, p, B / beams * H);
}

int gla_reorder_states(void* stream, int64_t count, void* const* tensors, const int64_t* row_bytes, int64_t requests, int64_t beams,
                       const int32_t* parents) {
  if (!parents || (count > 0 && (!tensors || !row_bytes))) return GLA_ERR_NULL_POINTER;
  if (count < 0 || requests <= 0 || beams <= 0) return GLA_ERR_BAD_DIMS;
  if (beams > 32) return GLA_ERR_UNSUPPORTED;
  for (int64_t i = 0; i < count; ++i) {
    if (!tensors[i]) return GLA_ERR_NULL_POINTER;
    if (row_bytes[i] <= 0) return GLA_ERR_BAD_DIMS;
  }
  // tensors by the widest access that their address and rows allow, RT of them a launch
  bool first = true;
  for (int unit = 16; unit; unit = unit == 16 ? 4 : unit == 4 ? 1 : 0) {
    beam::Tensors t{};
    t.K = (int)beams; t.parents = parents;
    unsigned int blocks = 0;
    const auto flush = [&]() -> int {
      if (!t.n) return GLA_OK;
      t.start[t.n] = blocks;
      t.count = first;
      first = false;
      const int s = unit == 16 ? beam::launch_reorder<uint4>((cudaStream_t)stream, t)
                    : unit == 4 ? beam::launch_reorder<uint32_t>((cudaStream_t)stream, t) : beam::launch_reorder<uint8_t>((cudaStream_t)stream, t);
      t.n = 0; blocks = 0;
      return s;
    };
    for (int64_t i = 0; i < count; ++i) {
      const uintptr_t both = (uintptr_t)tensors[i] | (uintptr_t)row_bytes[i];
      const int own = (both & 15) == 0 ? 16 : (both & 3) == 0 ? 4 : 1;
      if (own != unit) continue;
      const int64_t per = (row_bytes[i] / unit + beam::MNT - 1) / beam::MNT * requests;
      if (per > 1 << 30) return GLA_ERR_TOO_LARGE;
      if (t.n == beam::RT || (int64_t)blocks + per > 1 << 30) GLA_TRY(flush());
      t.p[t.n] = (uint8_t*)tensors[i];
      t.bytes[t.n] = row_bytes[i];
      t.start[t.n++] = blocks;
      blocks += (unsigned int)per;
    }
    GLA_TRY(flush());
  }
  return GLA_OK;
}

static int select_check(int64_t N, int64_t K, int64_t V, int64_t M, int dtype, int64_t pad) {
  if (N <= 0 || K <= 0 || V <= 0 || M <= 0 || M > K * V || pad < 0 || pad >= V) return GLA_ERR_BAD_DIMS;
  if (dtype != GLA_F32 && dtype != GLA_BF16) return GLA_ERR_UNSUPPORTED;
  if (K > 32 || M > 32) return GLA_ERR_UNSUPPORTED;
  if (N > GRID_MOST / 32 || V > 1 << 30) return GLA_ERR_TOO_LARGE;
  return GLA_OK;
}
static size_t select_bytes(int64_t N, int64_t K, int64_t M, int parts) {
  return align_up((size_t)(N * K * parts * M) * 8, 256) + align_up((size_t)(N * K * parts) * 16, 256);
}

size_t gla_beam_select_workspace_bytes(int64_t N, int64_t K, int64_t V, int64_t M, int dtype) {
  if (select_check(N, K, V, M, dtype, 0) != GLA_OK) return 0;
  int parts; int64_t part;
  beam::plan(N * K, V, (int)K, (int)M, &parts, &part);
  return select_bytes(N, K, M, parts);
}

int gla_beam_select(void* stream, int64_t N, int64_t K, int64_t V, int64_t M, int dtype, const void* logits, const float* scores,
                    const unsigned char* finished, int64_t pad_token, float* out_scores, int64_t* tokens, int32_t* parents, void* workspace,
                    size_t workspace_bytes) {
  if (!logits || !scores || !out_scores || !tokens || !parents) return GLA_ERR_NULL_POINTER;
  GLA_TRY(select_check(N, K, V, M, dtype, pad_token));
  if ((uintptr_t)logits % (dtype == GLA_BF16 ? 2 : 4)) return GLA_ERR_ALIGNMENT;
  beam::Select p{};
  p.logits = logits; p.scores = scores; p.finished = finished; p.V = V; p.K = (int)K; p.M = (int)M; p.bf = dtype == GLA_BF16; p.pad = pad_token;
  beam::plan(N * K, V, p.K, p.M, &p.parts, &p.part);
  if (!workspace || workspace_bytes < select_bytes(N, K, M, p.parts)) return GLA_ERR_WORKSPACE;
  if (!aligned16(workspace)) return GLA_ERR_ALIGNMENT;
  p.cand = (unsigned long long*)workspace;
  p.sums = (double2*)((char*)workspace + align_up((size_t)(N * K * p.parts * M) * 8, 256));
  p.out_scores = out_scores; p.tokens = (long long*)tokens; p.parents = parents;
  cudaStream_t st = (cudaStream_t)stream;
  {
    ProfScope ps("select_parts_kernel", st);
    const dim3 grid((unsigned)(N * K * p.parts));
    GLA_LAUNCHED(launch_overlapped(p.bf ? beam::select_parts_kernel<true> : beam::select_parts_kernel<false>, grid, dim3(beam::QNT), 0, st, p));
  }
  ProfScope ps("select_beams_kernel", st);
  GLA_LAUNCHED(launch_overlapped(beam::select_beams_kernel, dim3((unsigned)N), dim3(beam::BNT), 0, st, p));
  return GLA_OK;
}

}  // extern "C"
