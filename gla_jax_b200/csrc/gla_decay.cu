// Linear attention with one decay per head: what runs around the walks of gla_decay.cuh (runs of a sequence and their
// states, sums over shared heads, the gradient of the decays), forward and backward.
#include "gla_decay_fast.cuh"

namespace gla {
namespace decay {
namespace {

// The offsets that the walks go by: the first is 0, none falls or leaves [0, T].  Runs are found by a search over them, which
// only offsets that rise lead to every run once, and every row is some sequence's or behind the last.  One block, since the running
// maximum needs all before it; 3 us of a packed call.
__device__ unsigned int g_bad_offsets = 0;      // sequences whose offsets had to be changed
__global__ void __launch_bounds__(1024) offsets_kernel(const int* cu, int64_t nseq, int T, int* clean) {
  __shared__ int part[32];
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  int carry = 0;
  grid_dep_wait();
  grid_dep_launch();
  for (int64_t i0 = 0; i0 <= nseq; i0 += 1024) {
    const int64_t i = i0 + tid;
    int x = 0;
    if (i > 0 && i <= nseq) {
      const int a = cu[i - 1], b = cu[i];
      if (a < 0 || b < a || b > T || (i == 1 && a != 0)) atomicAdd(&g_bad_offsets, 1u);
      x = b < 0 ? 0 : b > T ? T : b;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d && y > x) x = y;
    }
    if (lane == 31) part[warp] = x;
    __syncthreads();
    int all = carry;
    for (int w = 0; w < 32; ++w) {
      if (w < warp && part[w] > x) x = part[w];
      if (part[w] > all) all = part[w];
    }
    if (carry > x) x = carry;
    if (i <= nseq) clean[i] = x;
    carry = all;
    __syncthreads();
  }
}

// The state that enters each run of a sequence, from what each run adds: four elements a thread, in place.  Four runs' sums
// are requested before the first is used.
__global__ void __launch_bounds__(128) entering_kernel(const Walk p) {
  const int64_t s = blockIdx.z, h = blockIdx.y, dd = (int64_t)p.kd * p.vd;
  const int e = (blockIdx.x * 128 + threadIdx.x) * 4;
  grid_dep_wait();
  grid_dep_launch();
  if (e >= dd) return;
  const int c = e / p.kd, k = e % p.kd;
  int64_t n = 1;
  const int64_t s0 = slot_of(p, s, 0, n);
  if (s0 + n > p.nslots) return;
  const int64_t at0 = (s * p.H + h) * dd + (int64_t)k * p.ik + (int64_t)c * p.ic;
  float4 x;
  x.x = ld_any(p.init, !p.init_f32, at0); x.y = ld_any(p.init, !p.init_f32, at0 + p.ik);
  x.z = ld_any(p.init, !p.init_f32, at0 + 2 * p.ik); x.w = ld_any(p.init, !p.init_f32, at0 + 3 * p.ik);
  const auto slot = [&](int64_t i) { return (s0 + (p.rev ? n - 1 - i : i)) * p.H + h; };
  for (int64_t i0 = 0; i0 < n; i0 += 4) {
    float4 add[4];
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j + 1 < n) {
        add[j] = *reinterpret_cast<const float4*>(p.seg_state + slot(i0 + j) * dd + e);
        f[j] = exp2f((float)p.seg_total[slot(i0 + j)]);
      }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < n) {
        *reinterpret_cast<float4*>(p.seg_state + slot(i0 + j) * dd + e) = x;
        if (i0 + j + 1 < n) {
          x.x = fmaf(f[j], x.x, add[j].x); x.y = fmaf(f[j], x.y, add[j].y);
          x.z = fmaf(f[j], x.z, add[j].z); x.w = fmaf(f[j], x.w, add[j].w);
        }
      }
  }
}

// out[row][hk][d] = sum over the heads that share hk of x[row][h][d], in order
template <typename T>
__global__ void __launch_bounds__(256) share_sum_kernel(const float* x, T* out, int64_t n, int share, int d) {
  const int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4;
  if (i >= n) return;
  const int64_t row = i / d, c = i % d;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j < share; ++j) {
    const float4 y = *reinterpret_cast<const float4*>(x + (row * share + j) * d + c);
    a.x += y.x; a.y += y.y; a.z += y.z; a.w += y.w;
  }
  st_f(out, i, a.x); st_f(out, i + 1, a.y); st_f(out, i + 2, a.z); st_f(out, i + 3, a.w);
}

// The pairs i >= t > j of a chunk of L tokens that gate t weighs, w_ij (q_i k_j)(do_i v_j) with float32 products: a block per chunk and
// head, into dg.  Sums of all of a token's pairs, as q dq - k dk has them, would leave these as differences of two sums whose
// errors then add up over the sequence (2 x 250 tokens, 2 heads of 64, gates of -3: 5e-6 of the norm against 6e-7; 2 us of 144).
// It runs beside the walks, whose blocks are few where time is short: it reads nothing of theirs, and ends after them (so that what
// follows in the stream finds both).
template <typename T, int L>
__global__ void __launch_bounds__(256) pairs_kernel(const Walk p, const T* dout, float* dg) {
  constexpr int R = L / 16, W = 32;                    // rows and columns of a thread, features at a time
  __shared__ float a[L][W + 1], b[L][W + 1], m[L][L + 1];
  __shared__ double gate[L];
  __shared__ float2 lam[L];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16, h = blockIdx.y;
  // the chunk's first token, and the run's tokens from there on
  int64_t t0, left;
  if (!p.cu) {
    const int64_t per = p.seg / L, i0 = blockIdx.x / per * p.seg % ((p.T + p.seg - 1) / p.seg * p.seg) + blockIdx.x % per * L;
    t0 = blockIdx.x / per / ((p.T + p.seg - 1) / p.seg) * p.T + i0;
    left = p.T - i0;
  } else {
    // sequence s, its run in cell c (see find_run) from token x on: chunks from number s + c + x / L on
    int64_t l = 0, u = p.nseq - 1;
    while (l < u) {
      const int64_t s = (l + u + 1) / 2;
      if (s + p.cu[s] / p.seg + p.cu[s] / L <= blockIdx.x) l = s; else u = s - 1;
    }
    const int64_t first = p.cu[l], end = p.cu[l + 1];
    int64_t c = (blockIdx.x - l) / (1 + p.seg / L);
    if (c < first / p.seg) c = first / p.seg;
    const int64_t x = c * p.seg > first ? c * p.seg : first, hi = (c + 1) * p.seg < end ? (c + 1) * p.seg : end;
    t0 = x + (blockIdx.x - l - c - x / L) * L;
    left = hi - t0;
  }
  if (left <= 0) {
    grid_dep_wait();
    return;
  }
  const int nv = left < L ? (int)left : L;
  if (tid < L) {
    const float x = tid < nv ? p.g[(t0 + tid) * p.gt + h] : 0.f;
    gate[tid] = (x < -200.f ? -200.f : x) * 1.4426950408889634;      // (as the walks take it)
  }
  __syncthreads();
  if (tid < L) {
    double v = 0.0;
    for (int i = 0; i <= tid; ++i) v += gate[i];
    const float hi = (float)v;
    lam[tid] = make_float2(hi, (float)(v - hi));
  }
  float s[2][R][R] = {};
  const int Hk = p.H / p.gk;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int d = which ? p.vd : p.kd, heads = which ? p.H : Hk, at = which ? h : h / p.gk;
    const T *x = which ? dout : (const T*)p.q, *y = which ? (const T*)p.v : (const T*)p.k;
    for (int d0 = 0; d0 < d; d0 += W) {
      __syncthreads();
      for (int i = tid; i < L * W; i += 256) {
        const int r = i / W, c = i % W;
        const int64_t e = ((t0 + r) * heads + at) * d + d0 + c;
        const bool in = r < nv && d0 + c < d;
        a[r][c] = in ? ld_f(x, e) : 0.f;
        b[r][c] = in ? ld_f(y, e) : 0.f;
      }
      __syncthreads();
#pragma unroll 8
      for (int c = 0; c < W; ++c) {
        float u[R], v[R];
#pragma unroll
        for (int i = 0; i < R; ++i) { u[i] = a[ty + 16 * i][c]; v[i] = b[tx + 16 * i][c]; }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
          for (int j = 0; j < R; ++j) s[which][i][j] = fmaf(u[i], v[j], s[which][i][j]);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < R; ++x)
#pragma unroll
    for (int y = 0; y < R; ++y) {
      const int i = ty + 16 * x, j = tx + 16 * y;
      const float2 li = lam[i], lj = lam[j];
      m[i][j] = j < i && i < nv ? s[0][x][y] * exp2f((li.x - lj.x) + (li.y - lj.y)) * s[1][x][y] : 0.f;
    }
  __syncthreads();
  if (tid < L) {                                       // row i: m[i][t] = the sum over j < t
    double sum = 0.0;
    for (int j = 0; j < L; ++j) {
      const float x = m[tid][j];
      m[tid][j] = (float)sum;
      sum += x;
    }
  }
  __syncthreads();
  if (tid < nv) {
    double sum = 0.0;
    for (int i = tid; i < nv; ++i) sum += m[i][tid];
    dg[(t0 + tid) * p.H + h] = (float)sum;
  }
  grid_dep_wait();
}

// dg_t = the chunk's pairs (in dg) + sum over i >= t of (a_i - b_i) + <S_T, dS_T>: a block per sequence and head, from the end, the
// running sum in 64 bits.
// The errors of a and b (float32 products, some 2^-23 of each, cut off to one side) add up.  At the first token the sum has to be
// <S_0, dS_0>: where these states are float32, what it is off by is taken back, in proportion to the magnitudes summed so far
// (10 x 16384 tokens, 8 heads of 64, soft gates: 6e-7 to 2.3e-6 of the norm without, 5e-7 to 8e-7 with it).
// A value or key that is not finite makes the sum not finite from there back, where dg reads neither: those tokens are summed
// from the other end, <S_0, dS_0> - sum over i < t.
struct Gate {
  const float *a, *b;               // [tiles][token][H]
  int tiles;
  const int* cu;
  int64_t T, nseq, rows;
  int H;
  const float* S;                   // [s][h] final state, float32
  const void *dS, *S0, *dS0;        // [s][h]: gradient of it, first state, gradient of that
  int state_f32;                    // their type
  int64_t dd;
  float* dg;
};
__global__ void __launch_bounds__(512) gate_grad_kernel(const Gate p) {
  __shared__ double part[16];
  __shared__ double carry;
  __shared__ unsigned long long bad;
  const int64_t s = blockIdx.x, h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  int64_t a = s * p.T, b = a + p.T;
  if (p.cu) {
    a = p.cu[s]; b = p.cu[s + 1];
    if (s == p.nseq - 1)
      for (int64_t t = b + tid; t < p.T; t += 512) p.dg[t * p.H + h] = 0.f;
  }
  double rate = 0.0;
  const auto term = [&](int64_t t, double* size) {
    double x = 0.0, y = 0.0;
    for (int i = 0; i < p.tiles; ++i) { x += p.a[(i * p.rows + t) * p.H + h]; y += p.b[(i * p.rows + t) * p.H + h]; }
    const double m = fabs(x) + fabs(y);
    if (size) *size = m;
    return rate == 0.0 ? x - y : x - y - rate * m;
  };
  const auto total = [&](double x) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    __syncthreads();
    if (lane == 0) part[warp] = x;
    __syncthreads();
    x = 0.0;
    for (int w = 0; w < 16; ++w) x += part[w];
    return x;
  };
  const int64_t at0 = (s * p.H + h) * p.dd;
  double dot = 0.0;
  for (int64_t e = tid; e < p.dd; e += 512) dot += (double)p.S[at0 + e] * ld_any(p.dS, !p.state_f32, at0 + e);
  dot = total(dot);
  const auto first = [&]() {
    double x = 0.0;
    for (int64_t e = tid; e < p.dd; e += 512) x += (double)ld_any(p.S0, !p.state_f32, at0 + e) * ld_any(p.dS0, !p.state_f32, at0 + e);
    return x;
  };
  if (p.state_f32) {
    double off = -first(), all = 0.0;
    for (int64_t t = a + tid; t < b; t += 512) {
      double m;
      off += term(t, &m);
      all += m;
    }
    off = total(off) + dot;
    all = total(all);
    // none where something is not finite, which has to stay with its tokens
    if (all > 0.0 && isfinite(off / all)) rate = off / all;
  }
  if (tid == 0) { carry = dot; bad = 0; }
  __syncthreads();
  for (int64_t end = b; end > a; end -= 512) {
    const int64_t t = end - 1 - tid;
    double x = t >= a ? term(t, nullptr) : 0.0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) part[warp] = x;
    __syncthreads();
    double before = carry;
    for (int w = 0; w < warp; ++w) before += part[w];
    x += before;
    if (t >= a) {
      if (isfinite(x)) p.dg[t * p.H + h] = (float)(x + p.dg[t * p.H + h]);
      else atomicMax(&bad, (unsigned long long)(t - a + 1));
    }
    __syncthreads();
    if (tid == 511) carry = x;
    __syncthreads();
  }
  const int64_t back = a + (int64_t)bad;                            // tokens before it are still to be done
  if (back == a) return;
  double before = total(first());
  for (int64_t t0 = a; t0 < back; t0 += 512) {
    const int64_t t = t0 + tid;
    double x = t < back ? term(t, nullptr) : 0.0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    const double prev = __shfl_up_sync(0xffffffffu, x, 1);
    if (lane == 31) part[warp] = x;
    __syncthreads();
    double y = before - (lane ? prev : 0.0);
    for (int w = 0; w < 16; ++w) {
      if (w < warp) y -= part[w];
      before -= part[w];
    }
    if (t < back) p.dg[t * p.H + h] = (float)(y + p.dg[t * p.H + h]);
    __syncthreads();
  }
}

int sm_count() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return sms[dev];
}

// Tokens of a run.  A walk has a block per run, head and tile of value columns; with fewer blocks than the device has
// SMs sequences are cut into runs, at the price of reading k and v twice and of two launches more
// (1155 tokens of 16 heads, 128 x 128: 46 us in runs of 384, 40 in runs of 256).  With blocks for half the SMs or more nothing is
// cut, whatever the lengths of packed sequences, which the host does not know.
int64_t run_tokens(int64_t T, int64_t nseq, int64_t H, int64_t vd, bool packed) {
  const int64_t blocks = H * ((vd + 127) / 128) * nseq, want = (int64_t)sm_count();
  int64_t n = packed ? want / (H * ((vd + 127) / 128)) : want / blocks;      // runs: of the packed axis, of each sequence
  if (blocks * 2 > want) n = 1;
  if (n > T / 128) n = T / 128;
  if (n <= 1) return align_up(T, 128);
  return align_up((T + n - 1) / n, 128);
}

}  // namespace

struct Dims {
  int64_t B, T, H, Hk, Dk, Dv, nseq;   // nseq > 0: packed, one axis of T tokens
  int bf, hid_f32;
  int64_t seqs() const { return nseq ? nseq : B; }
  int64_t rows() const { return B * T; }
  int64_t seg(int64_t vd) const { return run_tokens(T, seqs(), H, vd, nseq > 0); }
  int64_t slots(int64_t s) const { const int64_t n = (T + s - 1) / s; return nseq ? nseq + n : B * n; }
  bool cut(int64_t s) const { return s < T; }
  size_t seg_bytes(int64_t vd) const {
    const int64_t s = seg(vd);
    return cut(s) ? align_up((size_t)(slots(s) * H * Dk * Dv) * 4, 256) + align_up((size_t)(slots(s) * H) * 8, 256) : 0;
  }
};

static int walk(cudaStream_t st, int mode, const Walks& p, int n, bool out, const char* name) {
  switch (mode) {
    case M_ONE: return walk_one(st, p, n, out, name);
    case M_STATE: return walk_state(st, p, n, out, name);
    case M_FINE: return walk_fine(st, p, n, out, name);
    default: return walk_full(st, p, n, out, name);
  }
}
static int entering(cudaStream_t st, const Walk& p) {
  ProfScope ps("decay_entering_kernel", st);
  GLA_LAUNCHED(launch_overlapped(entering_kernel, dim3((unsigned)(((int64_t)p.kd * p.vd + 511) / 512), (unsigned)p.H, (unsigned)p.nseq), dim3(128), 0, st, p));
  return GLA_OK;
}
// Whole walks of one kind of sizes: the runs' sums and their entering states first where sequences are cut (ws: seg_bytes for
// each).
static int run_walks(cudaStream_t st, const Dims& d, int mode, Walks p, int n, void* ws, const char* first, const char* name) {
  for (int i = 0; i < n; ++i) {
    Walk& w = p.w[i];
    w.H = (int)d.H; w.T = d.T; w.nseq = d.seqs();
    w.seg = d.seg(w.vd);
    w.nslots = d.slots(w.seg);
    if (w.nslots > 2147483647LL) return GLA_ERR_TOO_LARGE;
    if (d.cut(w.seg)) {
      w.seg_state = (float*)((char*)ws + i * d.seg_bytes(w.vd));
      w.seg_total = (double*)((char*)w.seg_state + align_up((size_t)(w.nslots * d.H * d.Dk * d.Dv) * 4, 256));
    }
  }
  if (d.cut(p.w[0].seg)) {
    GLA_TRY(walk(st, mode, p, n, false, first));
    for (int i = 0; i < n; ++i) GLA_TRY(entering(st, p.w[i]));
  }
  return walk(st, mode, p, n, true, name);
}
static int run_walk(cudaStream_t st, const Dims& d, int mode, const Walk& p, void* ws, const char* first, const char* name) {
  Walks all{};
  all.w[0] = p;
  return run_walks(st, d, mode, all, 1, ws, first, name);
}

// ---- bf16, head sizes up to 128: the walks of gla_decay_tc.cuh and gla_decay_tcb.cuh ---------------------------------------------------------
static bool fast(const Dims& d) { return d.bf && d.Dk <= 128 && d.Dv <= 128; }
static size_t state_bytes(const Dims& d, int64_t n) { return align_up((size_t)(n * d.H * d.Dk * d.Dv) * 4, 256); }
// saved: final states in float32 | states that enter the runs (where sequences are cut) | offsets (where packed).  The first two for
// the walks below only: the others' backward makes its own, with more digits than their forward has.
static size_t saved_states(const Dims& d) {
  return fast(d) ? state_bytes(d, d.seqs()) + (d.cut(d.seg(128)) ? state_bytes(d, d.slots(d.seg(128))) : 0) : 0;
}
static size_t offset_bytes(const Dims& d) { return d.nseq ? align_up((size_t)(d.nseq + 1) * 4, 256) : 0; }
size_t saved_bytes(const Dims& d) { return saved_states(d) + offset_bytes(d); }
static size_t fast_totals(const Dims& d) { return align_up((size_t)(d.slots(d.seg(128)) * d.H) * 8, 256); }
static Walk fast_base(const Dims& d, const int* cu, const float* g, int64_t gt) {
  Walk p{};
  p.H = (int)d.H; p.T = d.T; p.nseq = d.seqs(); p.seg = d.seg(128); p.nslots = d.slots(p.seg);
  p.g = g; p.gt = gt; p.cu = cu;
  p.init_f32 = p.fin_f32 = d.hid_f32;
  return p;
}
static int fast_fwd(cudaStream_t st, const Dims& d, const int* cu, const void* h0, const float* g, int64_t gt, const void* v, const void* k,
                    const void* q, void* hf, void* out, void* saved, void* ws) {
  Walk p = fast_base(d, cu, g, gt);
  p.q = q; p.k = k; p.v = v;
  p.gq = p.gk = (int)(d.H / d.Hk); p.gv = 1;
  p.kd = (int)d.Dk; p.vd = (int)d.Dv;
  p.init = h0; p.ik = d.Dv; p.ic = 1;
  if (d.cut(p.seg)) {
    p.seg_total = (double*)ws;
    p.seg_state = (float*)(saved ? (char*)saved + state_bytes(d, d.seqs()) : (char*)ws + fast_totals(d));
    GLA_TRY(fast_walk(st, p, d.hid_f32 ? F_SUMS_STATE : F_SUMS, "decay_runs_kernel"));
    GLA_TRY(entering(st, p));
  }
  p.sk = 1; p.sc = d.Dk;
  p.fin = hf; p.fin32 = (float*)saved;
  p.out = out;
  return fast_walk(st, p, d.hid_f32 ? F_STATE : F_ONE, "decay_walk_kernel");
}
static int share_sum(cudaStream_t st, const Dims& d, const float* x, void* out);
static size_t fast_bwd_parts(const Dims& d, bool gate, size_t (&at)[4]) {
  const int64_t s = d.seg(128);
  at[0] = d.cut(s) ? fast_totals(d) : 0;
  at[1] = at[0] + (d.cut(s) ? state_bytes(d, d.slots(s)) : 0);
  at[2] = at[1] + (gate ? align_up((size_t)(WALK_COLS * d.rows() * d.H) * 4, 256) : 0);
  at[3] = at[2] + (d.H > d.Hk ? align_up((size_t)(d.rows() * d.H * d.Dk) * 4, 256) : 0);
  return at[3];
}
static int fast_bwd(cudaStream_t st, const Dims& d, const int* cu, const void* h0, const float* g, int64_t gt, const void* v, const void* k,
                    const void* q, const void* saved, const void* dhf, const void* dout, void* dh, float* dg, void* dv, void* dk, void* dq,
                    void* ws) {
  size_t at[4];
  fast_bwd_parts(d, dg != nullptr, at);
  const int share = (int)(d.H / d.Hk);
  float *a = (float*)((char*)ws + at[1]), *wide = (float*)((char*)ws + at[2]);
  Walk p = fast_base(d, cu, g, gt);
  const bool cut = d.cut(p.seg);
  float* runs = cut ? (float*)((char*)saved + state_bytes(d, d.seqs())) : nullptr;
  // dq: the forward's walk with roles exchanged, over the forward's states
  p.q = dout; p.k = v; p.v = k; p.gq = p.gk = 1; p.gv = share; p.kd = (int)d.Dv; p.vd = (int)d.Dk;
  p.init = h0; p.ik = 1; p.ic = d.Dv;
  p.seg_state = runs; p.sk = d.Dk; p.sc = 1;
  p.out = share > 1 ? (void*)wide : dq; p.out_f32 = share > 1;
  p.r = dg ? q : nullptr; p.gr = share; p.rdot = a;
  GLA_TRY(fast_walk(st, p, dg ? F_FINE : F_ONE, "decay_dq_kernel"));
  if (share > 1) GLA_TRY(share_sum(st, d, wide, dq));
  // the rest, backwards
  Back b{};
  b.w = fast_base(d, cu, g, gt);
  b.w.rev = 1;
  b.w.kd = (int)d.Dk; b.w.vd = (int)d.Dv;
  b.w.init = dhf; b.w.ik = d.Dv; b.w.ic = 1;
  if (cut) {
    b.w.seg_total = (double*)ws;
    b.w.seg_state = (float*)((char*)ws + at[0]);
    Walk r = b.w;
    r.k = q; r.v = dout; r.gk = share; r.gv = 1; r.gq = 1;
    GLA_TRY(fast_walk(st, r, F_SUMS, "decay_runs_kernel"));
    GLA_TRY(entering(st, r));
  }
  b.w.q = q; b.w.k = k; b.w.v = v; b.w.gq = b.w.gk = share; b.w.gv = 1;
  b.w.fin = dh;
  b.dout = dout; b.a = a; b.S_runs = runs; b.S_end = (const float*)saved; b.S_init = h0;
  b.dk = share > 1 ? (void*)wide : dk; b.dk_f32 = share > 1; b.dv = dv; b.dg = dg;
  GLA_TRY(fast_back(st, b, dg != nullptr));
  return share > 1 ? share_sum(st, d, wide, dk) : GLA_OK;
}

static size_t run_bytes(const Dims& d, bool saved) {
  if (!fast(d)) return d.seg_bytes(d.Dv);
  const int64_t s = d.seg(128);
  return d.cut(s) ? fast_totals(d) + (saved ? 0 : state_bytes(d, d.slots(s))) : 0;
}
size_t fwd_ws_bytes(const Dims& d, bool saved) { return run_bytes(d, saved) + (saved ? 0 : offset_bytes(d)); }
int fwd(cudaStream_t st, const Dims& d, const int* cu, const void* h0, const float* g, int64_t gt, const void* v, const void* k,
        const void* q, void* hf, void* out, void* saved, void* ws) {
  if (cu) {
    int* clean = (int*)(saved ? (char*)saved + saved_states(d) : (char*)ws + run_bytes(d, false));
    ProfScope ps("decay_offsets_kernel", st);
    GLA_LAUNCHED(launch_overlapped(offsets_kernel, dim3(1), dim3(1024), 0, st, cu, d.nseq, (int)d.T, clean));
    cu = clean;
  }
  if (fast(d)) return fast_fwd(st, d, cu, h0, g, gt, v, k, q, hf, out, saved, ws);
  Walk p{};
  p.q = q; p.k = k; p.v = v;
  p.gq = p.gk = (int)(d.H / d.Hk); p.gv = 1;
  p.kd = (int)d.Dk; p.vd = (int)d.Dv;
  p.g = g; p.gt = gt; p.cu = cu;
  p.init = h0; p.fin = hf; p.ik = d.Dv; p.ic = 1; p.init_f32 = p.fin_f32 = d.hid_f32;
  p.out = out; p.out_f32 = !d.bf;
  return run_walk(st, d, !d.bf ? M_FULL : d.hid_f32 ? M_STATE : M_ONE, p, ws, "decay_runs_kernel", "decay_walk_kernel");
}

// whether the three walks of a backward run the same kernel on the same runs, and few blocks each: then they run side by side
static bool alike(const Dims& d) {
  const auto kind = [](int64_t x) { return x <= 64 ? 0 : x <= 128 ? 1 : 2; };
  return d.H == d.Hk && kind(d.Dk) == kind(d.Dv) && column_tiles((int)d.Dk) == column_tiles((int)d.Dv) && d.seg(d.Dk) == d.seg(d.Dv);
}
static size_t bwd_parts(const Dims& d, bool gate, size_t (&at)[5]) {
  const int64_t share = d.H / d.Hk, tiles = (d.Dk + 127) / 128;
  const size_t seg = alike(d) ? 3 * d.seg_bytes(d.Dv) : d.seg_bytes(d.Dv) > d.seg_bytes(d.Dk) ? d.seg_bytes(d.Dv) : d.seg_bytes(d.Dk);
  const size_t dots = gate ? align_up((size_t)(tiles * d.rows() * d.H) * 4, 256) : 0;
  at[0] = seg;
  at[1] = at[0] + dots;
  at[2] = at[1] + dots;
  at[3] = at[2] + (share > 1 ? align_up((size_t)(d.rows() * d.H * d.Dk) * 4, 256) : 0);
  at[4] = at[3] + (gate ? state_bytes(d, d.seqs()) : 0);
  return at[4];
}
size_t bwd_ws_bytes(const Dims& d, bool gate) {
  size_t at[5], fa[4];
  return fast(d) ? fast_bwd_parts(d, gate, fa) : bwd_parts(d, gate, at);
}
static int share_sum(cudaStream_t st, const Dims& d, const float* x, void* out) {
  const int64_t n = d.rows() * d.Hk * d.Dk;
  const unsigned blocks = (unsigned)((n / 4 + 255) / 256);
  ProfScope ps("decay_share_sum_kernel", st);
  if (d.bf) share_sum_kernel<bf16><<<blocks, 256, 0, st>>>(x, (bf16*)out, n, (int)(d.H / d.Hk), (int)d.Dk);
  else share_sum_kernel<float><<<blocks, 256, 0, st>>>(x, (float*)out, n, (int)(d.H / d.Hk), (int)d.Dk);
  GLA_CHECK_LAUNCH();
  return GLA_OK;
}
// (the runs are those of the walks for dq and dk)
template <typename T, int L>
static int pairs(cudaStream_t st, const Dims& d, const int* cu, const float* g, int64_t gt, const void* v, const void* k, const void* q,
                 const void* dout, float* dg) {
  Walk p{};
  p.H = (int)d.H; p.T = d.T; p.nseq = d.seqs(); p.seg = d.seg(d.Dk); p.nslots = d.slots(p.seg);
  p.g = g; p.gt = gt; p.cu = cu;
  p.q = q; p.k = k; p.v = v; p.gk = (int)(d.H / d.Hk); p.kd = (int)d.Dk; p.vd = (int)d.Dv;
  const int64_t chunks = cu ? p.nslots + (d.T + L - 1) / L : p.nslots * (p.seg / L);
  if (chunks > 2147483647LL) return GLA_ERR_TOO_LARGE;
  ProfScope ps("decay_pairs_kernel", st);
  GLA_LAUNCHED(launch_overlapped(pairs_kernel<T, L>, dim3((unsigned)chunks, (unsigned)d.H), dim3(256), 0, st, p, (const T*)dout, dg));
  return GLA_OK;
}
int bwd(cudaStream_t st, const Dims& d, const int* cu, const void* h0, const float* g, int64_t gt, const void* v, const void* k,
        const void* q, const void* saved, const void* dhf, const void* dout, void* dh, float* dg, void* dv, void* dk, void* dq, void* ws) {
  if (cu) cu = (const int*)((const char*)saved + saved_states(d));
  if (fast(d)) return fast_bwd(st, d, cu, h0, g, gt, v, k, q, saved, dhf, dout, dh, dg, dv, dk, dq, ws);
  size_t at[5];
  bwd_parts(d, dg != nullptr, at);
  float *rq = (float*)((char*)ws + at[0]), *rk = (float*)((char*)ws + at[1]), *wide = (float*)((char*)ws + at[2]),
        *last = (float*)((char*)ws + at[3]);                    // the final states
  const int share = (int)(d.H / d.Hk), mode = d.bf ? M_FINE : M_FULL;
  Walks all{};
  Walk &p = all.w[0], &r = all.w[1], &t = all.w[2];
  p.g = g; p.gt = gt; p.cu = cu;
  p.init_f32 = p.fin_f32 = d.hid_f32;
  r = t = p;
  // dq, forwards over the states of the forward, transposed
  p.q = dout; p.k = v; p.v = k; p.gq = p.gk = 1; p.gv = share; p.kd = (int)d.Dv; p.vd = (int)d.Dk;
  p.init = h0; p.ik = 1; p.ic = d.Dv; p.fin32 = dg ? last : nullptr;
  p.out = share > 1 ? (void*)wide : dq; p.out_f32 = share > 1 || !d.bf;
  p.r = dg ? q : nullptr; p.gr = share; p.rdot = rq;
  // dk, backwards
  r.rev = 1;
  r.q = v; r.k = dout; r.v = q; r.gq = r.gk = 1; r.gv = share; r.kd = (int)d.Dv; r.vd = (int)d.Dk;
  r.init = dhf; r.ik = 1; r.ic = d.Dv;
  r.out = share > 1 ? (void*)wide : dk; r.out_f32 = share > 1 || !d.bf;
  r.r = dg ? k : nullptr; r.gr = share; r.rdot = rk;
  // dv and the gradient of the first state, backwards
  t.rev = 1;
  t.q = k; t.k = q; t.v = dout; t.gq = t.gk = share; t.gv = 1; t.kd = (int)d.Dk; t.vd = (int)d.Dv;
  t.init = dhf; t.ik = d.Dv; t.ic = 1; t.fin = dh;
  t.out = dv; t.out_f32 = !d.bf;
  if (alike(d)) {
    GLA_TRY(run_walks(st, d, mode, all, 3, ws, "decay_runs_kernel", "decay_grads_kernel"));
  } else {
    GLA_TRY(run_walk(st, d, mode, p, ws, "decay_runs_kernel", "decay_dq_kernel"));
    if (share > 1) GLA_TRY(share_sum(st, d, wide, dq));
    GLA_TRY(run_walk(st, d, mode, r, ws, "decay_runs_kernel", "decay_dk_kernel"));
    if (share > 1) GLA_TRY(share_sum(st, d, wide, dk));
    GLA_TRY(run_walk(st, d, mode, t, ws, "decay_runs_kernel", "decay_dv_kernel"));
  }
  if (dg) {
    const int s = d.bf ? pairs<bf16, Mode<M_FINE>::L>(st, d, cu, g, gt, v, k, q, dout, dg) : pairs<float, Mode<M_FULL>::L>(st, d, cu, g, gt, v, k, q, dout, dg);
    if (s != GLA_OK) return s;
    Gate w{};
    w.a = rq; w.b = rk; w.tiles = (int)((d.Dk + 127) / 128);
    w.cu = cu; w.T = d.T; w.nseq = d.seqs(); w.rows = d.rows(); w.H = (int)d.H;
    w.S = last; w.dS = dhf; w.S0 = h0; w.dS0 = dh; w.state_f32 = d.hid_f32; w.dd = d.Dk * d.Dv; w.dg = dg;
    ProfScope ps("decay_gate_grad_kernel", st);
    gate_grad_kernel<<<dim3((unsigned)w.nseq, (unsigned)d.H), 512, 0, st>>>(w);
    GLA_CHECK_LAUNCH();
  }
  return GLA_OK;
}
unsigned int read_bad_offsets() {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_bad_offsets, sizeof(v));
  return v;
}

// What the entry points share: sizes, types, alignment, workspace.
static int check(const Dims& d, int dtype, int hidden_dtype, const int* cu) {
  if (d.B <= 0 || d.T <= 0 || d.H <= 0 || d.Hk <= 0 || d.Dk <= 0 || d.Dv <= 0 || d.nseq < 0 || d.H % d.Hk) return GLA_ERR_BAD_DIMS;
  if ((d.nseq > 0) != (cu != nullptr) || (d.nseq > 0 && (d.B != 1 || d.T > 2147483647LL))) return GLA_ERR_BAD_DIMS;
  if ((dtype != GLA_F32 && dtype != GLA_BF16) || (hidden_dtype != GLA_F32 && hidden_dtype != dtype)) return GLA_ERR_UNSUPPORTED;
  if (d.Dk % 8 || d.Dv % 8 || d.Dk > 256 || d.Dv > 256) return GLA_ERR_UNSUPPORTED;
  // (sequences are cut into runs only where they are fewer than the SMs)
  if (d.H > 65535 / 4 || d.seqs() > 2147483647LL - 65536 || d.T > (int64_t)1 << 40) return GLA_ERR_TOO_LARGE;
  return GLA_OK;
}

}  // namespace decay
}  // namespace gla

using namespace gla;
using decay::Dims;

extern "C" {

static Dims dims_of(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, int hidden_dtype, int64_t nseq) {
  return Dims{B, T, H, Hk, Dk, Dv, nseq, dtype == GLA_BF16, hidden_dtype == GLA_F32};
}

size_t gla_decay_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, int hidden_dtype,
                                 int64_t nseq, int what) {
  const Dims d = dims_of(B, T, H, Hk, Dk, Dv, dtype, hidden_dtype, nseq);
  static const int some = 0;
  if (decay::check(d, dtype, hidden_dtype, nseq > 0 ? &some : nullptr) != GLA_OK) return 0;
  return what > 1 ? decay::bwd_ws_bytes(d, what == 3) : decay::fwd_ws_bytes(d, what == 1);
}

size_t gla_decay_saved_bytes(int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, int hidden_dtype, int64_t nseq) {
  const Dims d = dims_of(B, T, H, Hk, Dk, Dv, dtype, hidden_dtype, nseq);
  static const int some = 0;
  return decay::check(d, dtype, hidden_dtype, nseq > 0 ? &some : nullptr) == GLA_OK ? decay::saved_bytes(d) : 0;
}

int gla_decay_fwd(void* stream, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, int hidden_dtype,
                  int64_t nseq, const int32_t* cu_seqlens, const void* hidden_init, const float* log_decay, int per_token,
                  const void* value, const void* key, const void* query, void* hidden_final, void* out, void* saved,
                  void* workspace, size_t workspace_bytes) {
  if (!hidden_init || !log_decay || !value || !key || !query || !hidden_final || !out) return GLA_ERR_NULL_POINTER;
  const Dims d = dims_of(B, T, H, Hk, Dk, Dv, dtype, hidden_dtype, nseq);
  GLA_TRY(decay::check(d, dtype, hidden_dtype, cu_seqlens));
  for (const void* p : {value, key, query, (const void*)out})
    if (!aligned16(p)) return GLA_ERR_ALIGNMENT;
  const size_t need = decay::fwd_ws_bytes(d, saved != nullptr);
  if (!aligned16(saved)) return GLA_ERR_ALIGNMENT;
  if (need && (!workspace || workspace_bytes < need)) return GLA_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return GLA_ERR_ALIGNMENT;
  return decay::fwd((cudaStream_t)stream, d, cu_seqlens, hidden_init, log_decay, per_token ? H : 0, value, key, query, hidden_final, out,
                    saved, workspace);
}

int gla_decay_bwd(void* stream, int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype, int hidden_dtype,
                  int64_t nseq, const int32_t* cu_seqlens, const void* hidden_init, const float* log_decay, int per_token,
                  const void* value, const void* key, const void* query, const void* saved, const void* dhidden_final,
                  const void* dout, void* dhidden_init, float* dlog_decay, void* dvalue, void* dkey, void* dquery, void* workspace,
                  size_t workspace_bytes) {
  if (!hidden_init || !log_decay || !value || !key || !query || !dhidden_final || !dout || !dhidden_init || !dvalue || !dkey ||
      !dquery)
    return GLA_ERR_NULL_POINTER;
  const Dims d = dims_of(B, T, H, Hk, Dk, Dv, dtype, hidden_dtype, nseq);
  GLA_TRY(decay::check(d, dtype, hidden_dtype, cu_seqlens));
  if (!saved && decay::saved_bytes(d)) return GLA_ERR_NULL_POINTER;
  for (const void* p : {value, key, query, saved, dout, (const void*)dvalue, (const void*)dkey, (const void*)dquery})
    if (!aligned16(p)) return GLA_ERR_ALIGNMENT;
  const size_t need = decay::bwd_ws_bytes(d, dlog_decay != nullptr);
  if (need && (!workspace || workspace_bytes < need)) return GLA_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return GLA_ERR_ALIGNMENT;
  return decay::bwd((cudaStream_t)stream, d, cu_seqlens, hidden_init, log_decay, per_token ? H : 0, value, key, query, saved, dhidden_final,
                    dout, dhidden_init, dlog_decay, dvalue, dkey, dquery, workspace);
}

}  // extern "C"
