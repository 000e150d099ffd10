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

constexpr int TILE = 64;           // queries (keys) per workgroup, keys (queries) per pass of its loop
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
// the score in base 2; with a cap, `y` is the tanh (its derivative is 1 - y^2)
template <class T, bool CAP>
__device__ __forceinline__ float score(const Score& s, float dot, int ago, float& y) {
  float x = dot * s.mul;
  if (CAP) {
    y = cap_tanh<T>(x);
    x = y * s.cap;
  }
  return x - s.slope * (float)ago;
}

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
// A workgroup of four waves takes 64 queries of one head, a wave 16 of them, and walks the keys in
// tiles of 64 staged in LDS.  Scores are computed transposed (keys x queries), so a lane holds one
// query: its running maximum and sum are in-lane but for two shuffles, and the probabilities lie in
// registers as the B operand of out^T[dim][query] += V^T[dim][key] P^T[key][query].
template <class T, int D, bool CAP>
__global__ __launch_bounds__(256) void forward_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D);
  __shared__ __align__(16) T sK[TILE * LD];
  __shared__ __align__(16) T sV[TILE * LD];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int nt = (a.steps + TILE - 1) / TILE;
  const int q0 = (nt - 1 - (int)(blockIdx.x % nt)) * TILE;       // the longest ranges first
  const int eh = blockIdx.x / nt, h = eh % a.heads_q, e = eh / a.heads_q;
  const int hk = h / (a.heads_q / a.heads_k);
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int qi = q0 + 16 * w + m;
  const bool live = qi < n;
  const Score sc = score_of(a.scale, a.softcap, a.slopes, h);

  Frag<T> qf[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) qf[s] = Frag<T>{};
  if (live) {
    const T* qr = row<T>(a.q, e, qi, h);
#pragma unroll
    for (int s = 0; s < D / 32; ++s) qf[s] = load_run(qr, 32 * s, g);
  }
  const int32_t* begins = a.begins ? a.begins + (int64_t)e * a.steps : nullptr;
  const int begin = begins && live ? begins[qi] : 0;
  const int kend = min(q0 + TILE, n);
  const int kbeg = begins && q0 < n ? begins[q0] / TILE * TILE : 0;

  f32x4 o[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) o[d] = f32x4{0, 0, 0, 0};
  float mx = -INFINITY, sum = 0.0f;
  for (int k0 = kbeg; k0 < kend; k0 += TILE) {
    __syncthreads();
    stage<T, D, TILE>(sK, row<T>(a.k, e, k0, hk), a.k.step, kend - k0, tid, 256);
    stage<T, D, TILE>(sV, row<T>(a.v, e, k0, hk), a.v.step, kend - k0, tid, 256);
    __syncthreads();
    f32x4 s[TILE / 16];
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < TILE / 16; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) mma(s[t], load_run(sK + (16 * t + m) * LD, 32 * c, g), qf[c]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = k0 + 16 * t + 4 * g + r;
        float y;
        const float x = score<T, CAP>(sc, s[t][r], qi - j, y);
        s[t][r] = live && j <= qi && j >= begin ? x : -INFINITY;
        top = fmaxf(top, s[t][r]);
      }
    }
    top = fmaxf(mx, max_groups(top));
    // a query whose keys all lie in other tiles has nothing yet: exp2(-inf - 0) = 0
    const float base = top == -INFINITY ? 0.0f : top;
    const float old = __builtin_amdgcn_exp2f(mx - base);
    mx = top;
    float part = 0.0f;
#pragma unroll
    for (int t = 0; t < TILE / 16; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(s[t][r] - base);
        part += s[t][r];
      }
    sum = sum * old + part;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] *= old;
#pragma unroll
    for (int c = 0; c < TILE / 32; ++c) {
      const Frag<T> pf = round_frag<T>(join(s[2 * c], s[2 * c + 1]));
#pragma unroll
      for (int d = 0; d < D / 16; ++d) mma(o[d], load_col(sV, LD, 32 * c, 16 * d, lane), pf);
    }
  }
  sum = sum_groups(sum);
  if (qi >= a.steps) return;
  const float inv = live ? 1.0f / sum : 0.0f;
  T* out = row_out<T>(a.out, e, qi, h);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) store4(out + 16 * d + 4 * g, live ? o[d] * inv : f32x4{0, 0, 0, 0});
  if (a.lse && g == 0 && live) a.lse[((int64_t)e * a.heads_q + h) * a.steps + qi] = mx + log2f(sum);
}

// ---- backward ------------------------------------------------------------------------------
// dq: as the forward pass, with dp^T = V dout^T next to the scores and dq^T += K^T ds^T.  It also
// writes delta_i = dout_i.out_i for the pass over keys.
template <class T, int D, bool CAP>
__global__ __launch_bounds__(256) void backward_q_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D);
  __shared__ __align__(16) T sK[TILE * LD];
  __shared__ __align__(16) T sV[TILE * LD];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int nt = (a.steps + TILE - 1) / TILE;
  const int q0 = (nt - 1 - (int)(blockIdx.x % nt)) * TILE;
  const int eh = blockIdx.x / nt, h = eh % a.heads_q, e = eh / a.heads_q;
  const int hk = h / (a.heads_q / a.heads_k);
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int qi = q0 + 16 * w + m;
  const bool live = qi < n;
  const Score sc = score_of(a.scale, a.softcap, a.slopes, h);
  const int64_t at = ((int64_t)e * a.heads_q + h) * a.steps + qi;

  Frag<T> qf[D / 32], df[D / 32];
  float delta = 0.0f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) qf[s] = df[s] = Frag<T>{};
  if (live) {
    const T *qr = row<T>(a.q, e, qi, h), *dr = row<T>(a.dout, e, qi, h), *orow = row<T>(a.out, e, qi, h);
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      qf[s] = load_run(qr, 32 * s, g);
      df[s] = load_run(dr, 32 * s, g);
      const f32x8 x = widen(df[s]), y = widen(load_run(orow, 32 * s, g));
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(x[j], y[j], delta);
    }
  }
  delta = sum_groups(delta);
  if (live && g == 0) a.delta[at] = delta;
  const float lse = live ? a.lse[at] : 0.0f;
  const int32_t* begins = a.begins ? a.begins + (int64_t)e * a.steps : nullptr;
  const int begin = begins && live ? begins[qi] : 0;
  const int kend = min(q0 + TILE, n);
  const int kbeg = begins && q0 < n ? begins[q0] / TILE * TILE : 0;

  f32x4 dq[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) dq[d] = f32x4{0, 0, 0, 0};
  for (int k0 = kbeg; k0 < kend; k0 += TILE) {
    __syncthreads();
    stage<T, D, TILE>(sK, row<T>(a.k, e, k0, hk), a.k.step, kend - k0, tid, 256);
    stage<T, D, TILE>(sV, row<T>(a.v, e, k0, hk), a.v.step, kend - k0, tid, 256);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < TILE / 32; ++c) {
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
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = k0 + 16 * t + 4 * g + r;
          float y = 0.0f;
          const float x = score<T, CAP>(sc, s[r], qi - j, y);
          const float p = __builtin_amdgcn_exp2f(x - lse);
          float v = p * (dp[r] - delta);
          if (CAP) v *= 1.0f - y * y;
          ds[u][r] = live && j <= qi && j >= begin ? v : 0.0f;
        }
      }
      const Frag<T> f = round_frag<T>(join(ds[0], ds[1]));
#pragma unroll
      for (int d = 0; d < D / 16; ++d) mma(dq[d], load_col(sK, LD, 32 * c, 16 * d, lane), f);
    }
  }
  if (qi >= a.steps) return;
  T* out = row_out<T>(a.dq, e, qi, h);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) store4(out + 16 * d + 4 * g, live ? dq[d] * a.scale : f32x4{0, 0, 0, 0});
}

// dk, dv: a wave holds 16 keys and walks the queries that see them, of every query head that
// shares the key's head, so nothing is added across workgroups.
template <class T, int D, bool CAP>
__global__ __launch_bounds__(256) void backward_kv_kernel(bsg_attention a) {
  constexpr int LD = pitch<T>(D);
  __shared__ __align__(16) T sQ[TILE * LD];
  __shared__ __align__(16) T sD[TILE * LD];
  __shared__ __align__(16) float sLse[TILE], sDelta[TILE];
  __shared__ __align__(16) int sBegin[TILE];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int nt = (a.steps + TILE - 1) / TILE;
  const int k0 = (int)(blockIdx.x % nt) * TILE;                  // the longest ranges first
  const int eh = blockIdx.x / nt, hk = eh % a.heads_k, e = eh / a.heads_k;
  const int group = a.heads_q / a.heads_k;
  const int n = a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
  const int kj = k0 + 16 * w + m;
  const int32_t* begins = a.begins ? a.begins + (int64_t)e * a.steps : nullptr;

  Frag<T> kf[D / 32], vf[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) kf[s] = vf[s] = Frag<T>{};
  if (kj < n) {
    const T *kr = row<T>(a.k, e, kj, hk), *vr = row<T>(a.v, e, kj, hk);
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      kf[s] = load_run(kr, 32 * s, g);
      vf[s] = load_run(vr, 32 * s, g);
    }
  }
  f32x4 dk[D / 16], dv[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) dk[d] = dv[d] = f32x4{0, 0, 0, 0};
  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const Score sc = score_of(a.scale, a.softcap, a.slopes, h);
    const int64_t at = ((int64_t)e * a.heads_q + h) * a.steps;
    for (int q0 = k0; q0 < n; q0 += TILE) {
      if (begins && begins[q0] > k0 + TILE - 1) break;
      __syncthreads();
      stage<T, D, TILE>(sQ, row<T>(a.q, e, q0, h), a.q.step, n - q0, tid, 256);
      stage<T, D, TILE>(sD, row<T>(a.dout, e, q0, h), a.dout.step, n - q0, tid, 256);
      if (tid < TILE) {
        const bool on = q0 + tid < n;
        sLse[tid] = on ? a.lse[at + q0 + tid] : 0.0f;
        sDelta[tid] = on ? a.delta[at + q0 + tid] : 0.0f;
        // a query behind the last step sees no key: its range begins after every key
        sBegin[tid] = on ? (begins ? begins[q0 + tid] : 0) : 0x7fffffff;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < TILE / 32; ++c) {
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
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int l = 16 * t + 4 * g + r, i = q0 + l;
            float y = 0.0f;
            const float x = score<T, CAP>(sc, s[r], i - kj, y);
            const float p = __builtin_amdgcn_exp2f(x - sLse[l]);
            const bool on = kj <= i && kj >= sBegin[l];
            float v = p * (dp[r] - sDelta[l]);
            if (CAP) v *= 1.0f - y * y;
            ps[u][r] = on ? p : 0.0f;
            ds[u][r] = on ? v : 0.0f;
          }
        }
        const Frag<T> pf = round_frag<T>(join(ps[0], ps[1])), f = round_frag<T>(join(ds[0], ds[1]));
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          mma(dv[d], load_col(sD, LD, 32 * c, 16 * d, lane), pf);
          mma(dk[d], load_col(sQ, LD, 32 * c, 16 * d, lane), f);
        }
      }
    }
  }
  if (kj >= a.steps) return;
  const bool live = kj < n;
  T *ok = row_out<T>(a.dk, e, kj, hk), *ov = row_out<T>(a.dv, e, kj, hk);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    store4(ok + 16 * d + 4 * g, live ? dk[d] * a.scale : f32x4{0, 0, 0, 0});
    store4(ov + 16 * d + 4 * g, live ? dv[d] : f32x4{0, 0, 0, 0});
  }
}

// ---- acting --------------------------------------------------------------------------------
// A ring row (one slot's key or value of one head) is read by D / EPL lanes, EPL values (16 bytes)
// each, so a wave reads 64 EPL / D slots at once; each lane group keeps its own running maximum,
// sum and output for the G query heads that share the key, and they are joined at the end.
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
          s[u][i] = score<T, CAP>(sc[i], sum_lanes<LPR>(dot), ago[u], y);
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
        const float s = score<T, CAP>(sc[i], sum_lanes<LPR>(dot), 0, y);
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

// Long rings and few envs: `splits` workgroups of four waves share an item's slots and leave
// their maximum, sum and output in the workspace; a second launch joins them.
template <class T, int D, int G, bool CAP>
__global__ __launch_bounds__(256) void act_split_kernel(bsg_attention_act a, int splits, int span, int subs) {
  typedef Act<T, D, G, CAP> A;
  constexpr int EPL = A::EPL;
  __shared__ float sm[4][G], ss[4][G], sa[4][G][D];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int split = blockIdx.x % splits, ei = blockIdx.x / splits;
  const int items = a.heads_k * subs, item = ei % items, e = ei / items;
  const int group = a.heads_q / a.heads_k;
  const int hk = item / subs, sub = item % subs, h0 = hk * group + sub * G, heads = min(G, group - sub * G);
  const int n = steps_before(a, e), all = min(n, a.slots);
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

template <class T, int D>
__global__ __launch_bounds__(256) void act_join_kernel(bsg_attention_act a, int splits) {
  __shared__ float sacc[256], sbase[256];
  const int h = blockIdx.x % a.heads_q, e = blockIdx.x / a.heads_q;
  const float* p = static_cast<const float*>(a.work) + ((int64_t)e * a.heads_q + h) * splits * (D + 2);
  constexpr int P = 256 / D;                     // threads that share a value's splits
  const int c = threadIdx.x % D, part = threadIdx.x / D;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, p[s * (D + 2) + D]);   // split 0 saw the step itself
  float sum = 0.0f, acc = 0.0f;
  for (int s = part; s < splits; s += P) {
    const float f = __builtin_amdgcn_exp2f(p[s * (D + 2) + D] - top);
    sum += p[s * (D + 2) + D + 1] * f;
    acc += p[s * (D + 2) + c] * f;
  }
  sacc[threadIdx.x] = acc;
  sbase[threadIdx.x] = sum;
  __syncthreads();
  if (part == 0) {
    for (int i = 1; i < P; ++i) {
      acc += sacc[i * D + c];
      sum += sbase[i * D + c];
    }
    row_out<T>(a.out, e, 0, h)[c] = (T)(acc / sum);
  }
  if (h == 0 && threadIdx.x == 0) a.steps[e] = steps_after(steps_before(a, e));
}

// How an acting step is split: enough workgroups of four waves for every CU to hold four, none
// with fewer than 256 slots.  One workgroup per env (no second launch) where that is one split.
struct Plan { int g, subs, wpi, splits, span; };
Plan plan_of(const bsg_attention_act& a) {
  Plan p;
  const int group = a.heads_q / a.heads_k;
  p.g = group >= 4 ? 4 : group >= 2 ? 2 : 1;
  p.subs = (group + p.g - 1) / p.g;
  const int64_t items = (int64_t)a.heads_k * p.subs;
  p.wpi = items == 1 ? 4 : items == 2 ? 2 : 1;
  const int64_t want = (1024 + a.num_envs * items - 1) / (a.num_envs * items);
  const int64_t most = a.slots / 256;
  p.splits = (int)(want < most ? want : most);
  if (p.splits < 2) p.splits = 1;
  p.span = (a.slots + p.splits - 1) / p.splits;
  return p;
}

template <class T, int D, int G, bool CAP>
hipError_t act(const bsg_attention_act& a, const Plan& p, hipStream_t st) {
  if (p.splits == 1) {
    act_env_kernel<T, D, G, CAP><<<dim3(a.num_envs), dim3(256), 0, st>>>(a, p.wpi, p.subs);
  } else {
    act_split_kernel<T, D, G, CAP><<<dim3(a.num_envs * a.heads_k * p.subs * p.splits), dim3(256), 0, st>>>(
        a, p.splits, p.span, p.subs);
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

template <class T, int D, bool CAP>
hipError_t forward(const bsg_attention& a, hipStream_t st) {
  const int nt = (a.steps + TILE - 1) / TILE;
  if (a.begins && (a.first || a.window > 0))
    begins_kernel<<<dim3(a.num_envs), dim3(256), 0, st>>>(a.first, a.first_env, a.first_step, a.steps, a.window, a.begins);
  forward_kernel<T, D, CAP><<<dim3(a.num_envs * a.heads_q * nt), dim3(256), 0, st>>>(a);
  return hipGetLastError();
}
template <class T, int D, bool CAP>
hipError_t backward(const bsg_attention& a, hipStream_t st) {
  const int nt = (a.steps + TILE - 1) / TILE;
  backward_q_kernel<T, D, CAP><<<dim3(a.num_envs * a.heads_q * nt), dim3(256), 0, st>>>(a);
  backward_kv_kernel<T, D, CAP><<<dim3(a.num_envs * a.heads_k * nt), dim3(256), 0, st>>>(a);
  return hipGetLastError();
}
template <class T, int D>
hipError_t learn(const bsg_attention& a, bool back, hipStream_t st) {
  if (a.softcap > 0.0f) return back ? backward<T, D, true>(a, st) : forward<T, D, true>(a, st);
  return back ? backward<T, D, false>(a, st) : forward<T, D, false>(a, st);
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
int64_t attention_step_bytes(const bsg_attention_act& a) {
  const Plan p = plan_of(a);
  return p.splits == 1 ? 0 : (int64_t)a.num_envs * a.heads_q * p.splits * (a.dim + 2) * 4;
}

}  // namespace bsg
