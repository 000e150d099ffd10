// Attention of each RL step to the steps of its episode (bsg_attention_*, include/bsg.h): the
// learning form over rollouts with its gradients, and the acting form over a ring of the last
// steps' keys and values.
//
//   s_ij = scale q_i.k_j -> softcap tanh(s_ij / softcap) -> less slopes[h] (i - j)
//   p_ij = exp(s_ij - lse_i), lse_i = log sum_j exp(s_ij);  out_i = sum_j p_ij v_j
//   dp_ij = dout_i.v_j;  ds_ij = p_ij (dp_ij - dout_i.out_i) (1 - (s_ij / softcap)^2)
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij dout_i
// Step i sees j in [begin_i, i]; begin_i (its episode's first step, or the window's) never falls
// with i, so the keys of a tile of queries, and the queries of a tile of keys, are one range.
//
// Exponents are kept in base 2 (scores times log2 e): v_exp_f32 is a power of two.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "bsg_internal.h"
#include "bsg_mma.h"

namespace {

using namespace bsg::mma;

constexpr int TILE = BSG_ATTENTION_TILE;   // queries (keys) to a workgroup, keys (queries) to a turn of its loop
constexpr float LOG2E = 1.44269504088896340736f;

template <class T> __device__ __forceinline__ const T* row(const bsg_rows& x, int e, int t, int h) {
  return static_cast<const T*>(x.p) + e * x.env + t * x.step + h * x.head;
}
template <class T> __device__ __forceinline__ T* row_out(const bsg_rows& x, int e, int t, int h) {
  return static_cast<T*>(x.p) + e * x.env + t * x.step + h * x.head;
}

// tanh for the cap.  fp32 operands: the library's (a few ulp).  bf16: 1 - 2 / (1 + e^2x), whose
// absolute error of 2^-23 is far under the rounding that the scores' operands had.
template <class T> __device__ __forceinline__ float cap_tanh(float x);
template <> __device__ __forceinline__ float cap_tanh<float>(float x) { return tanhf(x); }
template <> __device__ __forceinline__ float cap_tanh<bf16>(float x) {
  return 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(2.0f * LOG2E * x));
}

struct Score {
  float mul;        // scale log2 e, or scale / softcap with a cap
  float cap;        // softcap log2 e
  float slope;      // slope log2 e
};
__device__ __forceinline__ Score score_of(float scale, float softcap, const float* slopes, int h) {
  Score s;
  s.mul = softcap > 0.0f ? scale / softcap : scale * LOG2E;
  s.cap = softcap * LOG2E;
  s.slope = slopes ? slopes[h] * LOG2E : 0.0f;
  return s;
}
// The score in base 2 plus `add` (ADD): the bias, -slope (i - j), or what of it varies inside a tile,
// which saves an instruction or two an element (2 envs x 4095 steps, dim 128 588 -> 576 us, 32 264 -> 249).
// With a cap, `y` is the tanh (its derivative is 1 - y^2).
template <class T, bool CAP, bool ADD>
__device__ __forceinline__ float score(const Score& s, float dot, float add, float& y) {
  if (CAP) {
    y = cap_tanh<T>(dot * s.mul);
    return ADD ? fmaf(y, s.cap, add) : y * s.cap;
  }
  return ADD ? fmaf(dot, s.mul, add) : dot * s.mul;
}

// Workgroups go to the eight XCDs in turn; each takes one contiguous eighth of the tiles, so that
// the tiles of a head, which read the same rows, share an L2.
__device__ __forceinline__ int swizzled(int b, int all) { return all % 8 ? b : b % 8 * (all / 8) + b / 8; }

// begins[e][t]: one workgroup per env walks its steps, 256 at a time; the last first step at or
// before t is the highest set bit of the wave's ballot up to its lane, or of an earlier wave's.
__global__ __launch_bounds__(256) void begins_kernel(const uint8_t* first, int64_t fe, int64_t ft, int T,
                                                     int window, int32_t* begins) {
  __shared__ int last[4];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int carry = 0;
  for (int t0 = 0; t0 < T; t0 += 256) {
    const int t = t0 + tid;
    const bool f = first && t < T && first[e * fe + t * ft] != 0;
    const unsigned long long all = __ballot(f);
    const unsigned long long up = all & (~0ull >> (63 - lane));
    if (lane == 0) last[w] = all ? t0 + 64 * w + 63 - __builtin_clzll(all) : -1;
    __syncthreads();
    int b = carry;
    for (int i = 0; i < 4; ++i) {
      const int l = last[i];
      if (i < w && l >= 0) b = l;
      if (l >= 0) carry = l;
    }
    if (up) b = t0 + 64 * w + 63 - __builtin_clzll(up);
    if (window > 0) b = max(b, t - window + 1);
    if (t < T) begins[(int64_t)e * T + t] = b;
    __syncthreads();
  }
}

// ---- forward -------------------------------------------------------------------------------
// A workgroup of four waves takes 64 queries of one head, a wave 16 of them, and walks the
// keys in tiles of 64, fetched one tile ahead through registers and shared in LDS.  Scores are
// computed transposed (keys x queries), so a lane holds one query: its running maximum and sum are
// in-lane but for two lane swaps, and the probabilities lie in registers as the B operand of
// out^T[dim][query] += V^T[dim][key] P^T[key][query].  (32 queries to a wave read LDS half as often
// but leave a SIMD half the waves to cover its loads: 605 against 581 us forward and backward at 2 envs x
// 4095 steps, dim 128; 459 against 370 us at dim 64.)
// Masks are only applied in tiles that an edge crosses.  2 x 4095 at dim 128: 165 us, 88 GFLOP of
// products at 530 TFLOP/s; three waves a SIMD, whose exponentials and products take turns; 256 x 300 at
// dim 64 with a cap: 44 us, two exponentials and a reciprocal a score.
template <class T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) void forward_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D), KT = TILE / 16;
  __shared__ __align__(16) T sK[TILE * LD];
  __shared__ __align__(16) T sV[TILE * LD];
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = (a.steps + TILE - 1) / TILE, id = swizzled(blockIdx.x, gridDim.x);
  const int q0 = (nt - 1 - id % nt) * TILE;                 // the longest ranges first
  const int eh = id / nt, h = eh % a.heads_q, e = eh / a.heads_q;
  const int hk = h / (a.heads_q / a.heads_k);
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int qw = q0 + 16 * w;                               // the wave's first query
  const Score sc = score_of(a.scale, a.softcap, a.slopes, h);
  const int32_t* begins = a.begins ? a.begins + (int64_t)e * a.steps : nullptr;

  Frag<T> qf[D / 32];
  const int qi = qw + m;
  // a query behind the last step reads the last one's row and is not written
  const int at = max(min(qi, n - 1), 0);
  const T* qr = row<T>(a.q, e, at, h);
#pragma unroll
  for (int s = 0; s < D / 32; ++s) qf[s] = load_run(qr, 32 * s, g);
  const int begin = begins ? begins[at] : 0;
  const int kend = min(q0 + TILE, n), kbeg = begins && q0 < n ? begins[q0] / TILE * TILE : 0;
  // what the wave's queries see: from the first one's begin; all of them from the last one's
  const int see_any = begins && qw < n ? begins[qw] : 0;
  const int see_all = begins && qw < n ? begins[min(qw + 16, n) - 1] : 0;

  f32x4 o[D / 16];
  float mx = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int d = 0; d < D / 16; ++d) o[d] = f32x4{0, 0, 0, 0};
  float along[KT][4];              // the bias along a tile's keys; the rest is the lane's and goes with the maximum
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) along[t][r] = BIAS ? sc.slope * (float)(16 * t + r) : 0.0f;
  const auto tile = [&](int k0, bool masked) {
    f32x4 s[KT];
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      // behind the wave's last query (fp32: worth a branch)
      if (sizeof(T) == 4 && k0 + 16 * t > qw + 15) {
        s[t] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        continue;
      }
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) mma(s[t], load_run(sK + (16 * t + m) * LD, 32 * c, g), qf[c]);
    }
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if (sizeof(T) == 4 && k0 + 16 * t > qw + 15) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y;
        s[t][r] = score<T, CAP, BIAS>(sc, s[t][r], along[t][r], y);
      }
      if (masked)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = k0 + 16 * t + 4 * g + r;
          s[t][r] = j <= qi && j >= begin ? s[t][r] : -INFINITY;
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][r]);
    }
    const float rest = BIAS ? -sc.slope * (float)(qi - k0 - 4 * g) : 0.0f;
    top = fmaxf(mx, max_groups(top + rest));
    // a query whose keys all lie in other tiles has nothing yet: exp2(-inf - 0) = 0
    const float now = top == -INFINITY ? 0.0f : top, old = __builtin_amdgcn_exp2f(mx - now), base = now - rest;
    mx = top;
    sum *= old;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - base);
        sum += s[t][r];
      }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] *= old;
#pragma unroll
    for (int c = 0; c < KT / 2; ++c) {
      if (sizeof(T) == 4 && k0 + 32 * c > qw + 15) continue;
      const Frag<T> pf = round_frag<T>(join(s[2 * c], s[2 * c + 1]));
#pragma unroll
      for (int d = 0; d < D / 16; ++d) mma(o[d], load_col(sV, LD, 32 * c, 16 * d, lane), pf);
    }
  };
  Fetch<T, TILE, D, 256> fk, fv;
  if (kbeg < kend) {
    fk.load(row<T>(a.k, e, kbeg, hk), a.k.step, kend - kbeg, tid);
    fv.load(row<T>(a.v, e, kbeg, hk), a.v.step, kend - kbeg, tid);
  }
  for (int k0 = kbeg; k0 < kend; k0 += TILE) {
    __syncthreads();
    fk.store(sK, kend - k0, tid);
    fv.store(sV, kend - k0, tid);
    if (k0 + TILE < kend) {
      fk.load(row<T>(a.k, e, k0 + TILE, hk), a.k.step, kend - k0 - TILE, tid);
      fv.load(row<T>(a.v, e, k0 + TILE, hk), a.v.step, kend - k0 - TILE, tid);
    }
    __syncthreads();
    if (qw >= n || k0 > qw + 15 || k0 + TILE <= see_any) continue;
    tile(k0, k0 + TILE - 1 > qw || k0 < see_all);
  }
  if (qi >= a.steps) return;
  const bool live = qi < n;
  const float all = sum_groups(sum), inv = live ? 1.0f / all : 0.0f;
  const int64_t to = ((int64_t)e * a.heads_q + h) * a.steps + qi;
  T* out = row_out<T>(a.out, e, qi, h);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const f32x4 x = live ? o[d] * inv : f32x4{0, 0, 0, 0};
    store4(out + 16 * d + 4 * g, x);
    if (sizeof(T) == 2 && a.out_rest) {                        // what the rounding left
      f32x4 rest;
#pragma unroll
      for (int r = 0; r < 4; ++r) rest[r] = x[r] - (float)(T)x[r];
      store4(static_cast<T*>(a.out_rest) + to * D + 16 * d + 4 * g, rest);
    }
  }
  if (a.lse && g == 0 && live) a.lse[to] = mx + log2f(all);
}

// ---- backward ------------------------------------------------------------------------------
// p and ds of 16 keys (rows 4g + r) and a lane's query, or of 16 queries and a lane's key; `add`: the
// bias less lse.  Where an edge crosses the tile, on(r) says which are seen.
template <class T, bool CAP, class On>
__device__ __forceinline__ void p_and_ds(const Score& sc, const f32x4& add, const f32x4& delta, const f32x4& s, const f32x4& dp,
                                         bool masked, On on, f32x4& p, f32x4& ds) {
  f32x4 x, y = {0, 0, 0, 0};
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float t = 0.0f;
    x[r] = score<T, CAP, true>(sc, s[r], add[r], t);
    y[r] = t;
  }
  if (masked)
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = on(r) ? x[r] : -INFINITY;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    p[r] = __builtin_amdgcn_exp2f(x[r]);
    ds[r] = p[r] * (dp[r] - delta[r]);
    if (CAP) ds[r] *= fmaf(-y[r], y[r], 1.0f);
  }
}

// Rollouts of one tile (64 steps): one workgroup per env and key head computes all three
// gradients from p and ds computed once.  A wave holds 16 queries for p, ds and dq (and delta, from
// the whole row of p and dp, so that the rounded out is not needed); p and ds then go to LDS, where V
// and K were, and the wave takes 16 keys, whose dk and dv it adds up over the query heads that share
// them.  512 envs x 50 steps, 4 heads, fp32, dim 64: 68 us (by the passes below 122), bound by fp32 matrix
// instructions.
template <class T, int D>
struct Short {
  static constexpr int N = D > TILE ? D : TILE, LD = pitch<T>(D), PD = pitch<T>(TILE);
  T q[TILE * LD], go[TILE * LD];
  T k[TILE * pitch<T>(N)], v[TILE * pitch<T>(N)];                // then ds and p, [query][key]
};
template <class T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256) void backward_short_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D), PD = pitch<T>(TILE), KT = TILE / 16;
  __shared__ __align__(16) Short<T, D> x;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % a.heads_k, e = blockIdx.x / a.heads_k, group = a.heads_q / a.heads_k;
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int own = 16 * w + m;
  const bool live = own < n;
  const int begin = live && a.begins ? a.begins[(int64_t)e * a.steps + own] : 0;
  f32x4 dk[D / 16], dv[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) dk[d] = dv[d] = f32x4{0, 0, 0, 0};
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const Score sc = score_of(a.scale, a.softcap, a.slopes, h);
    const float lse = live ? a.lse[((int64_t)e * a.heads_q + h) * a.steps + own] : 0.0f;
    Fetch<T, TILE, D, 256> fk, fv, fq, fd;
    if (n > 0) {
      fk.load(row<T>(a.k, e, 0, hk), a.k.step, n, tid);
      fq.load(row<T>(a.q, e, 0, h), a.q.step, n, tid);
      fv.load(row<T>(a.v, e, 0, hk), a.v.step, n, tid);
      fd.load(row<T>(a.dout, e, 0, h), a.dout.step, n, tid);
    }
    __syncthreads();               // the head before is done with
    if (n > 0) {
      fk.store(x.k, n, tid);
      fq.store(x.q, n, tid);
      fv.store(x.v, n, tid);
      fd.store(x.go, n, tid);
    }
    __syncthreads();
    // rows of keys, a lane's query; the tiles of keys behind the wave's queries stay zero
    f32x4 p[KT], ds[KT], dq[D / 16];
#pragma unroll
    for (int t = 0; t < KT; ++t) p[t] = ds[t] = f32x4{0, 0, 0, 0};
    if (16 * w < n) {
      f32x4 dp[KT];
      float delta = 0.0f;
#pragma unroll
      for (int t = 0; t < KT; ++t)
        if (t <= w) {
          f32x4 s = {0, 0, 0, 0};
          dp[t] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            mma(s, load_run(x.k + (16 * t + m) * LD, 32 * c, g), load_run(x.q + own * LD, 32 * c, g));
            mma(dp[t], load_run(x.v + (16 * t + m) * LD, 32 * c, g), load_run(x.go + own * LD, 32 * c, g));
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * t + 4 * g + r;
            float y = 0.0f;
            const float z = score<T, CAP, BIAS>(sc, s[r], -sc.slope * (float)(own - j), y);
            const bool on = live && j <= own && j >= begin;
            p[t][r] = on ? __builtin_amdgcn_exp2f(z - lse) : 0.0f;
            ds[t][r] = CAP ? p[t][r] * fmaf(-y, y, 1.0f) : p[t][r];
            delta = fmaf(p[t][r], dp[t][r], delta);
          }
        }
      delta = sum_groups(delta);
#pragma unroll
      for (int t = 0; t < KT; ++t)
        if (t <= w) ds[t] *= dp[t] - delta;
    }
    __syncthreads();               // V is done with: p takes its place
#pragma unroll
    for (int t = 0; t < KT; ++t) store4(x.v + own * PD + 16 * t + 4 * g, p[t]);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) dq[d] = f32x4{0, 0, 0, 0};
    if (16 * w < n) {
#pragma unroll
      for (int c = 0; c < KT / 2; ++c)
        if (2 * c <= w) {
          const Frag<T> f = round_frag<T>(join(ds[2 * c], ds[2 * c + 1]));
#pragma unroll
          for (int d = 0; d < D / 16; ++d) mma(dq[d], load_col(x.k, LD, 32 * c, 16 * d, lane), f);
        }
    }
    __syncthreads();               // K is done with: ds takes its place
#pragma unroll
    for (int t = 0; t < KT; ++t) store4(x.k + own * PD + 16 * t + 4 * g, ds[t]);
    if (own < a.steps) {
      T* out = row_out<T>(a.dq, e, own, h);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) store4(out + 16 * d + 4 * g, live ? dq[d] * a.scale : f32x4{0, 0, 0, 0});
    }
    __syncthreads();
    // a lane's key: the queries from the wave's tile on
#pragma unroll
    for (int c = 0; c < KT / 2; ++c)
      if (2 * c + 1 >= w && 32 * c < n) {
        const Frag<T> pf = load_col(x.v, PD, 32 * c, 16 * w, lane), f = load_col(x.k, PD, 32 * c, 16 * w, lane);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          mma(dv[d], load_col(x.go, LD, 32 * c, 16 * d, lane), pf);
          mma(dk[d], load_col(x.q, LD, 32 * c, 16 * d, lane), f);
        }
      }
  }
  if (own >= a.steps) return;
  T *ok = row_out<T>(a.dk, e, own, hk), *ov = row_out<T>(a.dv, e, own, hk);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    store4(ok + 16 * d + 4 * g, live ? dk[d] * a.scale : f32x4{0, 0, 0, 0});
    store4(ov + 16 * d + 4 * g, live ? dv[d] : f32x4{0, 0, 0, 0});
  }
}

// Longer rollouts.  bf16: three waves a SIMD where the registers hold them without spilling (256 envs x
// 300 steps, dim 64 with a cap 168 -> 163 us, 512 envs 284 -> 262; dq at dim 128 with a cap spills: 290 -> 300).
// dq: as the forward pass, with dp^T = V dout^T next to the scores and
// dq^T += K^T ds^T.  It also writes delta_i = dout_i.out_i for the pass over keys; out is taken
// with what its rounding left, else delta would carry that rounding into every ds of the row.
// 2 x 4095 at dim 128: 190 us, 132 GFLOP (700 TFLOP/s).
template <class T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && !(D == 128 && CAP) ? 3 : 1)) void backward_q_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D), KT = TILE / 16;
  __shared__ __align__(16) T sK[TILE * LD];
  __shared__ __align__(16) T sV[TILE * LD];
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = (a.steps + TILE - 1) / TILE, id = swizzled(blockIdx.x, gridDim.x);
  const int q0 = (nt - 1 - id % nt) * TILE;
  const int eh = id / nt, h = eh % a.heads_q, e = eh / a.heads_q;
  const int hk = h / (a.heads_q / a.heads_k);
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int qw = q0 + 16 * w;
  const Score sc = score_of(a.scale, a.softcap, a.slopes, h);
  const int64_t base = ((int64_t)e * a.heads_q + h) * a.steps;
  const int32_t* begins = a.begins ? a.begins + (int64_t)e * a.steps : nullptr;

  Frag<T> qf[D / 32], df[D / 32];
  const int qi = qw + m, at = max(min(qi, n - 1), 0);            // a query behind the last step: the last one's row
  const T *qr = row<T>(a.q, e, at, h), *dr = row<T>(a.dout, e, at, h), *orow = row<T>(a.out, e, at, h);
  const T* rest = static_cast<const T*>(a.out_rest) + (base + at) * D;
  float x = 0.0f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    qf[s] = load_run(qr, 32 * s, g);
    df[s] = load_run(dr, 32 * s, g);
    const f32x8 u = widen(df[s]);
    f32x8 v = widen(load_run(orow, 32 * s, g));
    if (sizeof(T) == 2) v += widen(load_run(rest, 32 * s, g));
#pragma unroll
    for (int j = 0; j < 8; ++j) x = fmaf(u[j], v[j], x);
  }
  const float delta = sum_groups(x), lse = n > 0 ? a.lse[base + at] : 0.0f;
  if (g == 0 && qi < n) a.delta[base + qi] = delta;
  const int begin = begins ? begins[at] : 0;
  const int kend = min(q0 + TILE, n), kbeg = begins && q0 < n ? begins[q0] / TILE * TILE : 0;
  const int see_any = begins && qw < n ? begins[qw] : 0;
  const int see_all = begins && qw < n ? begins[min(qw + 16, n) - 1] : 0;

  f32x4 dq[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) dq[d] = f32x4{0, 0, 0, 0};
  const auto tile = [&](int k0, bool masked) {
    const float rest = (BIAS ? -sc.slope * (float)(qi - k0 - 4 * g) : 0.0f) - lse;
#pragma unroll
    for (int c = 0; c < KT / 2; ++c) {
      if (sizeof(T) == 4 && k0 + 32 * c > qw + 15) continue;
      f32x4 ds[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = 2 * c + u;
        f32x4 s = {0, 0, 0, 0}, dp = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          mma(s, load_run(sK + (16 * t + m) * LD, 32 * x, g), qf[x]);
          mma(dp, load_run(sV + (16 * t + m) * LD, 32 * x, g), df[x]);
        }
        f32x4 p, add;
        const f32x4 dl = {delta, delta, delta, delta};
#pragma unroll
        for (int r = 0; r < 4; ++r) add[r] = BIAS ? fmaf(sc.slope, (float)(16 * t + r), rest) : rest;
        const auto on = [&](int r) {
          const int j = k0 + 16 * t + 4 * g + r;
          return j <= qi && j >= begin;
        };
        p_and_ds<T, CAP>(sc, add, dl, s, dp, masked, on, p, ds[u]);
      }
      const Frag<T> f = round_frag<T>(join(ds[0], ds[1]));
#pragma unroll
      for (int d = 0; d < D / 16; ++d) mma(dq[d], load_col(sK, LD, 32 * c, 16 * d, lane), f);
    }
  };
  Fetch<T, TILE, D, 256> fk, fv;
  if (kbeg < kend) {
    fk.load(row<T>(a.k, e, kbeg, hk), a.k.step, kend - kbeg, tid);
    fv.load(row<T>(a.v, e, kbeg, hk), a.v.step, kend - kbeg, tid);
  }
  for (int k0 = kbeg; k0 < kend; k0 += TILE) {
    __syncthreads();
    fk.store(sK, kend - k0, tid);
    fv.store(sV, kend - k0, tid);
    if (k0 + TILE < kend) {
      fk.load(row<T>(a.k, e, k0 + TILE, hk), a.k.step, kend - k0 - TILE, tid);
      fv.load(row<T>(a.v, e, k0 + TILE, hk), a.v.step, kend - k0 - TILE, tid);
    }
    __syncthreads();
    if (qw >= n || k0 > qw + 15 || k0 + TILE <= see_any) continue;
    tile(k0, k0 + TILE - 1 > qw || k0 < see_all);
  }
  if (qi >= a.steps) return;
  const bool live = qi < n;
  T* out = row_out<T>(a.dq, e, qi, h);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) store4(out + 16 * d + 4 * g, live ? dq[d] * a.scale : f32x4{0, 0, 0, 0});
}

// dk, dv: a wave holds 16 keys and walks the queries that see them, in tiles of 64 fetched one
// ahead.  A workgroup does so for every query head that shares the key's head, so that nothing is
// added across workgroups; or, where that leaves CUs idle (`parts`), for one of them, into fp32
// partial sums that add_parts_kernel adds.  2 x 4095 at dim 128: 245 us, 177 GFLOP (720 TFLOP/s): two
// accumulators of 16 keys x 128 and two operand rows leave two waves a SIMD.
template <class T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && D <= 64 ? 3 : 1)) void backward_kv_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D), QT = TILE / 16;
  __shared__ __align__(16) T sQ[TILE * LD];
  __shared__ __align__(16) T sD[TILE * LD];
  __shared__ __align__(16) float sLse[TILE], sDelta[TILE];
  __shared__ __align__(16) int sBegin[TILE];
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = (a.steps + TILE - 1) / TILE, id = swizzled(blockIdx.x, gridDim.x);
  const int k0 = id % nt * TILE;                            // the longest ranges first
  const int group = a.heads_q / a.heads_k, eh = id / nt;
  const bool split = a.parts != nullptr;
  const int h0 = split ? eh % a.heads_q : eh % a.heads_k * group, h1 = split ? h0 + 1 : h0 + group;
  const int hk = h0 / group, e = split ? eh / a.heads_q : eh / a.heads_k;
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int kw = k0 + 16 * w;                               // the wave's first key
  const int32_t* begins = a.begins ? a.begins + (int64_t)e * a.steps : nullptr;

  Frag<T> kf[D / 32], vf[D / 32];
  f32x4 dk[D / 16], dv[D / 16];
  const int kj = kw + m, at = max(min(kj, n - 1), 0);
  const T *kr = row<T>(a.k, e, at, hk), *vr = row<T>(a.v, e, at, hk);
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    kf[s] = load_run(kr, 32 * s, g);
    vf[s] = load_run(vr, 32 * s, g);
  }
#pragma unroll
  for (int d = 0; d < D / 16; ++d) dk[d] = dv[d] = f32x4{0, 0, 0, 0};
  // the queries that see one of the keys end with the tile where the next episode (window) has begun:
  // begins never falls, so halving finds it
  int qend = n;
  if (begins && k0 < n) {
    int some = 0, none = (n - k0 + TILE - 1) / TILE;             // tiles from k0 that see, that do not
    while (none - some > 1) {
      const int t = (some + none) / 2;
      if (begins[k0 + t * TILE] > k0 + TILE - 1) none = t;
      else some = t;
    }
    qend = min(n, k0 + none * TILE);
  }

  Fetch<T, TILE, D, 256> fq, fd;
  float flse = 0.0f, fdelta = 0.0f;
  int fbegin = 0;
  const auto fetch = [&](int h, int q0) {
    fq.load(row<T>(a.q, e, q0, h), a.q.step, n - q0, tid);
    fd.load(row<T>(a.dout, e, q0, h), a.dout.step, n - q0, tid);
    const int64_t at = ((int64_t)e * a.heads_q + h) * a.steps;
    const int q = min(q0 + tid % TILE, n - 1);
    flse = a.lse[at + q];
    fdelta = a.delta[at + q];
    fbegin = begins ? begins[q] : 0;
  };
  if (k0 < qend) fetch(h0, k0);
  for (int h = h0; h < h1; ++h) {
    const Score sc = score_of(a.scale, a.softcap, a.slopes, h);
    const auto tile = [&](int q0, bool masked) {
      const float rest = BIAS ? sc.slope * (float)(kj - q0) : 0.0f;
#pragma unroll
      for (int c = 0; c < QT / 2; ++c) {
        if (sizeof(T) == 4 && q0 + 32 * c + 31 < kw) continue;   // before the wave's first key
        f32x4 ps[2], ds[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int t = 2 * c + u;
          f32x4 s = {0, 0, 0, 0}, dp = {0, 0, 0, 0};
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            mma(s, load_run(sQ + (16 * t + m) * LD, 32 * x, g), kf[x]);
            mma(dp, load_run(sD + (16 * t + m) * LD, 32 * x, g), vf[x]);
          }
          const f32x4 add = rest - *reinterpret_cast<const f32x4*>(&sLse[16 * t + 4 * g]);
          const f32x4 delta = *reinterpret_cast<const f32x4*>(&sDelta[16 * t + 4 * g]);
          const auto on = [&](int r) {
            const int l = 16 * t + 4 * g + r;
            return kj <= q0 + l && kj >= sBegin[l];
          };
          p_and_ds<T, CAP>(sc, add, delta, s, dp, masked, on, ps[u], ds[u]);
        }
        const Frag<T> pf = round_frag<T>(join(ps[0], ps[1])), f = round_frag<T>(join(ds[0], ds[1]));
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          mma(dv[d], load_col(sD, LD, 32 * c, 16 * d, lane), pf);
          mma(dk[d], load_col(sQ, LD, 32 * c, 16 * d, lane), f);
        }
      }
    };
    for (int q0 = k0; q0 < qend; q0 += TILE) {
      __syncthreads();
      fq.store(sQ, n - q0, tid);
      fd.store(sD, n - q0, tid);
      if (tid < TILE) {
        sLse[tid] = BIAS ? fmaf(sc.slope, (float)tid, flse) : flse;   // with the bias along the tile
        sDelta[tid] = fdelta;
        // a query behind the last step sees no key: its range begins after every key
        sBegin[tid] = q0 + tid < n ? fbegin : 0x7fffffff;
      }
      if (q0 + TILE < qend) fetch(h, q0 + TILE);
      else if (h + 1 < h1) fetch(h + 1, k0);
      __syncthreads();
      if (kw >= n || q0 + TILE - 1 < kw || sBegin[0] > kw + 15) continue;
      // unless every query of the tile sees every key of the wave
      tile(q0, kw + 15 > q0 || sBegin[TILE - 1] > kw);
    }
  }
  if (kj >= a.steps) return;
  const bool live = kj < n;
  if (split) {
    float* to = a.parts + (((int64_t)e * a.heads_q + h0) * a.steps + kj) * 2 * D;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      store4(to + 16 * d + 4 * g, live ? dk[d] * a.scale : f32x4{0, 0, 0, 0});
      store4(to + D + 16 * d + 4 * g, live ? dv[d] : f32x4{0, 0, 0, 0});
    }
  } else {
    T *ok = row_out<T>(a.dk, e, kj, hk), *ov = row_out<T>(a.dv, e, kj, hk);
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      store4(ok + 16 * d + 4 * g, live ? dk[d] * a.scale : f32x4{0, 0, 0, 0});
      store4(ov + 16 * d + 4 * g, live ? dv[d] : f32x4{0, 0, 0, 0});
    }
  }
}
// one thread per four values of a key's dk and dv: the query heads' parts in their order
template <class T, int D>
__global__ __launch_bounds__(256) void add_parts_kernel(bsg_attention a, int64_t all) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  const int c = (int)(i % (D / 2)) * 4, group = a.heads_q / a.heads_k;
  const int t = (int)(i / (D / 2) % a.steps);
  const int64_t eh = i / (D / 2) / a.steps;
  const int hk = (int)(eh % a.heads_k), e = (int)(eh / a.heads_k);
  f32x4 x = {0, 0, 0, 0};
  for (int h = hk * group; h < (hk + 1) * group; ++h)
    x += *reinterpret_cast<const f32x4*>(a.parts + (((int64_t)e * a.heads_q + h) * a.steps + t) * 2 * D + c);
  if (c < D) store4(row_out<T>(a.dk, e, t, hk) + c, x);
  else store4(row_out<T>(a.dv, e, t, hk) + c - D, x);
}

// ---- acting --------------------------------------------------------------------------------
// A ring row (one slot's key or value of one head) is read by D / EPL lanes, EPL values (16 bytes)
// each, so a wave reads 64 EPL / D slots at once; each lane group keeps its own running maximum,
// sum and output for the G query heads that share the key, and they are joined at the end.  The ring is
// read once and bounds the call: 4096 envs x 300 slots 120 us with full rings (629 MB), 3 x 30001 23 us
// with half full ones and 5 us for the join.
constexpr int UNROLL = 4;          // slots per lane group in flight

template <int N> __device__ __forceinline__ float sum_lanes(float x) {   // over groups of N lanes
  // quad_perm xor 1, xor 2, then row_half_mirror / row_mirror: lanes that hold equal sums by then
  if (N > 1) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xf, 0xf, true));
  if (N > 2) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xf, 0xf, true));
  if (N > 4) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xf, 0xf, true));
  if (N > 8) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xf, 0xf, true));
  if (N > 16) x += __shfl_xor(x, 16);
  return x;
}

template <class T, int EPL> __device__ __forceinline__ void load_vec(float* x, const T* p);
template <> __device__ __forceinline__ void load_vec<float, 4>(float* x, const float* p) {
  const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = v[i];
}
template <> __device__ __forceinline__ void load_vec<bf16, 8>(float* x, const bf16* p) {
  const f32x8 v = widen(*reinterpret_cast<const bf16x8*>(p));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = v[i];
}

// What a wave has seen: per query head the maximum and sum (base 2), and the lane's EPL outputs.
template <int G, int EPL> struct Seen { float mx[G], sum[G], acc[G][EPL]; };

template <class T, int D, int G, bool CAP>
struct Act {
  static constexpr int EPL = Vec<T>::n, LPR = D / EPL, SPW = 64 / LPR;

  // joins what lane groups `step` apart have seen
  static __device__ __forceinline__ void join_lanes(Seen<G, EPL>& x) {
#pragma unroll
    for (int step = LPR; step < 64; step *= 2)
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const float om = __shfl_xor(x.mx[q], step), os = __shfl_xor(x.sum[q], step);
        const float top = fmaxf(x.mx[q], om), base = top == -INFINITY ? 0.0f : top;
        const float a = __builtin_amdgcn_exp2f(x.mx[q] - base), b = __builtin_amdgcn_exp2f(om - base);
        x.mx[q] = top;
        x.sum[q] = x.sum[q] * a + os * b;
#pragma unroll
        for (int i = 0; i < EPL; ++i) x.acc[q][i] = x.acc[q][i] * a + __shfl_xor(x.acc[q][i], step) * b;
      }
  }

  // slots [lo, hi) of the ring of head (e, hk), `part` of `parts` waves; the current step, which
  // its slot may not hold yet, is taken from k and v by part 0 of the first range
  static __device__ __forceinline__ void see(Seen<G, EPL>& x, const bsg_attention_act& a, int e, int hk,
                                             int h0, int heads, int n, int lo, int hi, int part, int parts,
                                             bool own, int lane) {
    const int S = a.slots, cur = n % S, grp = lane / LPR, d0 = lane % LPR * EPL;
    float q[G][EPL];
    Score sc[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int h = h0 + min(i, heads - 1);     // a head that is not there repeats the last one
      load_vec<T, EPL>(q[i], row<T>(a.q, e, 0, h) + d0);
      sc[i] = score_of(a.scale, a.softcap, a.slopes, h);
      x.mx[i] = -INFINITY;
      x.sum[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) x.acc[i][j] = 0.0f;
    }
    const int64_t base = ((int64_t)e * a.heads_k + hk) * S;
    const T* kc = static_cast<const T*>(a.k_cache) + base * D + d0;
    const T* vc = static_cast<const T*>(a.v_cache) + base * D + d0;
    for (int s0 = lo + part * SPW * UNROLL; s0 < hi; s0 += parts * SPW * UNROLL) {
      float kx[UNROLL][EPL], vx[UNROLL][EPL], s[UNROLL][G];
      bool on[UNROLL];
      int ago[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int slot = s0 + u * SPW + grp;
        on[u] = slot < hi && slot != cur;
        ago[u] = cur - slot + (slot > cur ? S : 0);
        const int64_t at = (int64_t)min(slot, hi - 1) * D;
        load_vec<T, EPL>(kx[u], kc + at);
        load_vec<T, EPL>(vx[u], vc + at);
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int i = 0; i < G; ++i) {
          float dot = 0.0f;
#pragma unroll
          for (int j = 0; j < EPL; ++j) dot = fmaf(q[i][j], kx[u][j], dot);
          float y;
          s[u][i] = score<T, CAP, true>(sc[i], sum_lanes<LPR>(dot), -sc[i].slope * (float)ago[u], y);
          s[u][i] = on[u] ? s[u][i] : -INFINITY;
        }
      // what a masked slot holds is not even multiplied by zero: it may be anything
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int j = 0; j < EPL; ++j) vx[u][j] = on[u] ? vx[u][j] : 0.0f;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        float top = x.mx[i];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) top = fmaxf(top, s[u][i]);
        const float base2 = top == -INFINITY ? 0.0f : top;
        const float old = __builtin_amdgcn_exp2f(x.mx[i] - base2);
        x.mx[i] = top;
        x.sum[i] *= old;
#pragma unroll
        for (int j = 0; j < EPL; ++j) x.acc[i][j] *= old;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const float p = __builtin_amdgcn_exp2f(s[u][i] - base2);
          x.sum[i] += p;
#pragma unroll
          for (int j = 0; j < EPL; ++j) x.acc[i][j] = fmaf(p, vx[u][j], x.acc[i][j]);
        }
      }
    }
    if (own && grp == 0) {
      float kx[EPL], vx[EPL];
      load_vec<T, EPL>(kx, row<T>(a.k, e, 0, hk) + d0);
      load_vec<T, EPL>(vx, row<T>(a.v, e, 0, hk) + d0);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        float dot = 0.0f, y;
#pragma unroll
        for (int j = 0; j < EPL; ++j) dot = fmaf(q[i][j], kx[j], dot);
        const float s = score<T, CAP, true>(sc[i], sum_lanes<LPR>(dot), 0.0f, y);
        const float top = fmaxf(x.mx[i], s);
        const float old = __builtin_amdgcn_exp2f(x.mx[i] - top), p = __builtin_amdgcn_exp2f(s - top);
        x.mx[i] = top;
        x.sum[i] = x.sum[i] * old + p;
#pragma unroll
        for (int j = 0; j < EPL; ++j) x.acc[i][j] = x.acc[i][j] * old + p * vx[j];
      }
    }
    join_lanes(x);
  }

  // the step's key and value into their slot (lane group 0 of one wave); nobody reads it there
  static __device__ __forceinline__ void append(const bsg_attention_act& a, int e, int hk, int n, int lane) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    if (lane >= LPR) return;
    const int64_t at = (((int64_t)e * a.heads_k + hk) * a.slots + n % a.slots) * D + lane * EPL;
    *reinterpret_cast<u32x4*>(static_cast<T*>(a.k_cache) + at) =
        *reinterpret_cast<const u32x4*>(row<T>(a.k, e, 0, hk) + lane * EPL);
    *reinterpret_cast<u32x4*>(static_cast<T*>(a.v_cache) + at) =
        *reinterpret_cast<const u32x4*>(row<T>(a.v, e, 0, hk) + lane * EPL);
  }
};

__device__ __forceinline__ int steps_before(const bsg_attention_act& a, int e) {
  const int n = a.first && a.first[e * a.first_env] ? 0 : a.steps[e];
  return n < 0 ? 0 : n;
}
__device__ __forceinline__ int steps_after(int n) { return n == 0x7fffffff ? n : n + 1; }

template <class T, int EPL> __device__ __forceinline__ void store_vec(T* p, const float* x, float mul) {
#pragma unroll
  for (int i = 0; i < EPL; i += 4)
    store4(p + i, f32x4{x[i] * mul, x[i + 1] * mul, x[i + 2] * mul, x[i + 3] * mul});
}

// One workgroup per env: its waves share the items (a key head and up to G of its query heads),
// `wpi` waves to an item.  The env's step count is read by all and advanced at the end by one.
template <class T, int D, int G, bool CAP>
__global__ __launch_bounds__(256) void act_env_kernel(bsg_attention_act a, int wpi, int subs) {
  typedef Act<T, D, G, CAP> A;
  constexpr int EPL = A::EPL;
  __shared__ float sm[4][G], ss[4][G], sa[4][G][D];
  const int e = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = steps_before(a, e), group = a.heads_q / a.heads_k;
  const int items = a.heads_k * subs, stride = 4 / wpi, part = w % wpi;
  const int hi = min(n, a.slots);
  for (int i0 = 0; i0 < items; i0 += stride) {
    const int item = i0 + w / wpi;
    if (item < items) {
      const int hk = item / subs, sub = item % subs, h0 = hk * group + sub * G, heads = min(G, group - sub * G);
      Seen<G, EPL> x;
      A::see(x, a, e, hk, h0, heads, n, 0, hi, part, wpi, part == 0, lane);
      if (sub == 0 && part == 0) A::append(a, e, hk, n, lane);
      if (wpi == 1) {
        if (lane < A::LPR)
#pragma unroll
          for (int i = 0; i < G; ++i)
            if (i < heads) store_vec<T, EPL>(row_out<T>(a.out, e, 0, h0 + i) + lane * EPL, x.acc[i], 1.0f / x.sum[i]);
      } else if (lane < A::LPR) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
          if (lane == 0) {
            sm[w][i] = x.mx[i];
            ss[w][i] = x.sum[i];
          }
#pragma unroll
          for (int j = 0; j < EPL; ++j) sa[w][i][lane * EPL + j] = x.acc[i][j];
        }
      }
    }
    if (wpi > 1) {
      __syncthreads();
      if (item < items) {
        const int hk = item / subs, sub = item % subs, h0 = hk * group + sub * G, heads = min(G, group - sub * G);
        const int w0 = w - part;
        for (int d = part * 64 + lane; d < heads * D; d += wpi * 64) {
          const int i = d / D, c = d % D;
          float top = -INFINITY, sum = 0.0f, acc = 0.0f;
          for (int p = 0; p < wpi; ++p) top = fmaxf(top, sm[w0 + p][i]);   // part 0 saw the step itself
          for (int p = 0; p < wpi; ++p) {
            const float f = __builtin_amdgcn_exp2f(sm[w0 + p][i] - top);
            sum += ss[w0 + p][i] * f;
            acc += sa[w0 + p][i][c] * f;
          }
          row_out<T>(a.out, e, 0, h0 + i)[c] = (T)(acc / sum);
        }
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) a.steps[e] = steps_after(n);
}

// Long rings and few envs: `splits` workgroups of four waves share the slots that an item holds, in
// even parts, and leave their maximum, sum and output in the workspace; a second launch joins them.
template <class T, int D, int G, bool CAP>
__global__ __launch_bounds__(256) void act_split_kernel(bsg_attention_act a, int splits, int subs) {
  typedef Act<T, D, G, CAP> A;
  constexpr int EPL = A::EPL;
  __shared__ float sm[4][G], ss[4][G], sa[4][G][D];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int split = blockIdx.x % splits, ei = blockIdx.x / splits;
  const int items = a.heads_k * subs, item = ei % items, e = ei / items;
  const int group = a.heads_q / a.heads_k;
  const int hk = item / subs, sub = item % subs, h0 = hk * group + sub * G, heads = min(G, group - sub * G);
  const int n = steps_before(a, e), all = min(n, a.slots), span = (all + splits - 1) / splits;
  const int lo = min(split * span, all), hi = min(lo + span, all);
  Seen<G, EPL> x;
  A::see(x, a, e, hk, h0, heads, n, lo, hi, w, 4, split == 0 && w == 0, lane);
  if (split == 0 && sub == 0 && w == 0) A::append(a, e, hk, n, lane);
  if (lane < A::LPR)
#pragma unroll
    for (int i = 0; i < G; ++i) {
      if (lane == 0) {
        sm[w][i] = x.mx[i];
        ss[w][i] = x.sum[i];
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) sa[w][i][lane * EPL + j] = x.acc[i][j];
    }
  __syncthreads();
  float* work = static_cast<float*>(a.work);
  for (int d = threadIdx.x; d < heads * D; d += 256) {
    const int i = d / D, c = d % D;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (int p = 0; p < 4; ++p) top = fmaxf(top, sm[p][i]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int p = 0; p < 4; ++p) {
      const float f = __builtin_amdgcn_exp2f(sm[p][i] - base);
      sum += ss[p][i] * f;
      acc += sa[p][i][c] * f;
    }
    float* o = work + (((int64_t)e * a.heads_q + h0 + i) * splits + split) * (D + 2);
    o[c] = acc;
    if (c == 0) {
      o[D] = top;
      o[D + 1] = sum;
    }
  }
}

// A workgroup per env and query head: a split's weight per thread, then the values by rows of D threads.
constexpr int MAX_SPLITS = 256;
template <class T, int D>
__global__ __launch_bounds__(256) void act_join_kernel(bsg_attention_act a, int splits) {
  __shared__ float weight[MAX_SPLITS], acc[256], top4[4], sum4[4];
  const int h = blockIdx.x % a.heads_q, e = blockIdx.x / a.heads_q, tid = threadIdx.x;
  const float* p = static_cast<const float*>(a.work) + ((int64_t)e * a.heads_q + h) * splits * (D + 2);
  const float mx = tid < splits ? p[tid * (D + 2) + D] : -INFINITY, sm = tid < splits ? p[tid * (D + 2) + D + 1] : 0.0f;
  float top = mx;
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (tid % 64 == 0) top4[tid / 64] = top;
  __syncthreads();
  top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));   // split 0 saw the step itself
  const float f = __builtin_amdgcn_exp2f(mx - top);
  weight[tid] = f;
  float sum = sm * f;
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) sum += __shfl_xor(sum, d);
  if (tid % 64 == 0) sum4[tid / 64] = sum;
  __syncthreads();
  constexpr int P = 256 / D;                     // threads that share a value's splits
  const int c = tid % D, part = tid / D;
  float x = 0.0f;
#pragma unroll 8
  for (int s = part; s < splits; s += P) x = fmaf(p[s * (D + 2) + c], weight[s], x);
  acc[tid] = x;
  __syncthreads();
  if (part == 0) {
#pragma unroll
    for (int i = 1; i < P; ++i) x += acc[i * D + c];
    row_out<T>(a.out, e, 0, h)[c] = (T)(x / ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3])));
  }
  if (h == 0 && tid == 0) a.steps[e] = steps_after(steps_before(a, e));
}

// How an acting step is split: two workgroups of four waves to a CU, which is what its registers
// hold (one more makes a second round of a few), none with fewer than 256 slots of a full ring.  One
// workgroup per env (no second launch) where that is one split.
struct Plan { int g, subs, wpi, splits; };
Plan plan_of(const bsg_attention_act& a) {
  Plan p;
  const int group = a.heads_q / a.heads_k;
  p.g = group >= 4 ? 4 : group >= 2 ? 2 : 1;
  p.subs = (group + p.g - 1) / p.g;
  const int64_t items = (int64_t)a.heads_k * p.subs;
  p.wpi = items == 1 ? 4 : items == 2 ? 2 : 1;
  const int64_t want = 512 / (a.num_envs * items);
  const int64_t most = a.slots / 256;
  p.splits = (int)(want < most ? want : most);
  if (p.splits > MAX_SPLITS) p.splits = MAX_SPLITS;
  if (p.splits < 2) p.splits = 1;
  return p;
}

template <class T, int D, int G, bool CAP>
hipError_t act(const bsg_attention_act& a, const Plan& p, hipStream_t st) {
  if (p.splits == 1) {
    act_env_kernel<T, D, G, CAP><<<dim3(a.num_envs), dim3(256), 0, st>>>(a, p.wpi, p.subs);
  } else {
    act_split_kernel<T, D, G, CAP><<<dim3(a.num_envs * a.heads_k * p.subs * p.splits), dim3(256), 0, st>>>(
        a, p.splits, p.subs);
    act_join_kernel<T, D><<<dim3(a.num_envs * a.heads_q), dim3(256), 0, st>>>(a, p.splits);
  }
  return hipGetLastError();
}
template <class T, int D>
hipError_t act(const bsg_attention_act& a, hipStream_t st) {
  const Plan p = plan_of(a);
  const bool cap = a.softcap > 0.0f;
  if (p.g == 4) return cap ? act<T, D, 4, true>(a, p, st) : act<T, D, 4, false>(a, p, st);
  if (p.g == 2) return cap ? act<T, D, 2, true>(a, p, st) : act<T, D, 2, false>(a, p, st);
  return cap ? act<T, D, 1, true>(a, p, st) : act<T, D, 1, false>(a, p, st);
}

template <class T, int D, bool CAP, bool BIAS>
hipError_t forward(const bsg_attention& a, hipStream_t st) {
  const int nt = (a.steps + TILE - 1) / TILE;
  if (a.begins)
    begins_kernel<<<dim3(a.num_envs), dim3(256), 0, st>>>(a.first, a.first_env, a.first_step, a.steps, a.window, a.begins);
  forward_kernel<T, D, CAP, BIAS><<<dim3(a.num_envs * a.heads_q * nt), dim3(256), 0, st>>>(a);
  return hipGetLastError();
}
template <class T, int D, bool CAP, bool BIAS>
hipError_t backward(const bsg_attention& a, hipStream_t st) {
  if (a.steps <= TILE) {
    backward_short_kernel<T, D, CAP, BIAS><<<dim3(a.num_envs * a.heads_k), dim3(256), 0, st>>>(a);
    return hipGetLastError();
  }
  const int nt = (a.steps + TILE - 1) / TILE;
  backward_q_kernel<T, D, CAP, BIAS><<<dim3(a.num_envs * a.heads_q * nt), dim3(256), 0, st>>>(a);
  const int heads = a.parts ? a.heads_q : a.heads_k;
  backward_kv_kernel<T, D, CAP, BIAS><<<dim3(a.num_envs * heads * nt), dim3(256), 0, st>>>(a);
  if (a.parts) {
    const int64_t all = (int64_t)a.num_envs * a.heads_k * a.steps * (D / 2);
    add_parts_kernel<T, D><<<dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st>>>(a, all);
  }
  return hipGetLastError();
}
template <class T, int D, bool CAP, bool BIAS>
hipError_t learn(const bsg_attention& a, bool back, hipStream_t st) {
  return back ? backward<T, D, CAP, BIAS>(a, st) : forward<T, D, CAP, BIAS>(a, st);
}
template <class T, int D>
hipError_t learn(const bsg_attention& a, bool back, hipStream_t st) {
  if (a.softcap > 0.0f) return a.slopes ? learn<T, D, true, true>(a, back, st) : learn<T, D, true, false>(a, back, st);
  return a.slopes ? learn<T, D, false, true>(a, back, st) : learn<T, D, false, false>(a, back, st);
}
template <class T>
hipError_t learn(const bsg_attention& a, bool back, hipStream_t st) {
  return a.dim == 32 ? learn<T, 32>(a, back, st) : a.dim == 64 ? learn<T, 64>(a, back, st) : learn<T, 128>(a, back, st);
}
template <class T>
hipError_t act(const bsg_attention_act& a, hipStream_t st) {
  return a.dim == 32 ? act<T, 32>(a, st) : a.dim == 64 ? act<T, 64>(a, st) : act<T, 128>(a, st);
}

}  // namespace

namespace bsg {

// Shapes, strides and pointers are validated by the bsg_attention_* entry points (bsg_abi.cpp).
hipError_t launch_attention(const bsg_attention& a, bool back, hipStream_t st) {
  return a.dtype == BSG_BF16 ? learn<mma::bf16>(a, back, st) : learn<float>(a, back, st);
}
hipError_t launch_attention_step(const bsg_attention_act& a, hipStream_t st) {
  return a.dtype == BSG_BF16 ? act<mma::bf16>(a, st) : act<float>(a, st);
}
// Parts by query head are wanted where key tiles alone give fewer than four workgroups to a CU.
bool attention_wants_parts(const bsg_attention& a) {
  if (a.heads_q == a.heads_k || a.steps <= TILE) return false;
  return (int64_t)a.num_envs * a.heads_k * ((a.steps + TILE - 1) / TILE) < 1024;
}
int64_t attention_step_bytes(const bsg_attention_act& a) {
  const Plan p = plan_of(a);
  return p.splits == 1 ? 0 : (int64_t)a.num_envs * a.heads_q * p.splits * (a.dim + 2) * 4;
}

}  // namespace bsg
