// The gated delta rule (bsg_delta_*, include/bsg.h): the learning form over rollouts with its
// gradients, and the acting form of one RL step.
//
// Per env and value head, with alpha_t = e^{g_t} and a state S[dim_k][dim_v]:
//   w_t = v_t - alpha_t S^T k_t,   S <- alpha_t S + beta_t k_t w_t^T,   o_t = scale S^T q_t
// A chunk of C = 64 steps is solved at once.  With c_i = sum of g up to i inside the chunk,
// G_ij = e^{c_i - c_j} where i and j belong to one episode (else 0), S the state before the chunk,
//   N_ij = G_ij k_i.k_j (j < i),   P_ij = scale G_ij q_i.k_j (j <= i),
//   in_i = e^{c_i} where no episode began up to i (else 0),  out_j = e^{c_C - c_j} where none
//   began after j (else 0),  across = e^{c_C} where none began:
//   (I + N diag(beta)) W = V - in (K S),   U = beta W,
//   O = scale in (Q S) + P U,              S' = across S + K^T (out U)
// The unit lower triangular system is solved in blocks of 16 steps: the diagonal blocks are
// inverted, the rest are products.
// Backward, with X' the gradient of X and D the gradient of S':
//   U' = P^T O' + out (K D),  (I + N^T diag(beta)) M = U',  L = beta M = V',  beta'_i = w_i.m_i
//   gradient of S = across D + Q^T (scale in O') - K^T (in L)
//   q'_i  = scale (in_i S o'_i + sum_{j<=i} (o'_i.u_j) G_ij k_j)
//   kr'_i = -in_i S l_i - sum_{j<i} (l_i.u_j) G_ij k_j                  (k as it reads S)
//   kw'_j = out_j D u_j + scale sum_{i>=j} (o'_i.u_j) G_ij q_i - sum_{i>j} (l_i.u_j) G_ij k_i
//   k' = kr' + kw';  c'_i = q_i.q'_i + k_i.kr'_i - k_i.kw'_i, and the chunk's last step gets
//   across <S, D> + sum_j k_j.(out_j D u_j);  g'_t = the sum of c'_i from t to its episode's end.
//
// c is summed in double and kept as two floats, so that the difference of two of them is exact to
// the difference's own rounding however far both have run down.  States, W and M are fp32; where
// they meet bf16 operands they are split into bf16 parts (bsg_mma.h): three (24 bits) on every
// path that leads into a state, which stays fp32 to the caller, two (2^-17) on those that end in a
// bf16 output.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "bsg_internal.h"
#include "bsg_mma.h"

namespace {

using namespace bsg::mma;

constexpr int C = BSG_DELTA_CHUNK;
constexpr int AP = C + 4;          // row pitch of the C x C matrices in LDS
constexpr int IP = 20;             // ... of the 16 x 16 inverses
constexpr float LOWEST = -1e5f;    // the least log decay: its exponential is 0

template <class T> __device__ __forceinline__ const T* row(const bsg_rows& x, int e, int t, int h) {
  return static_cast<const T*>(x.p) + e * x.env + t * x.step + h * x.head;
}
template <class T> __device__ __forceinline__ T* row_out(const bsg_rows& x, int e, int t, int h) {
  return static_cast<T*>(x.p) + e * x.env + t * x.step + h * x.head;
}
__device__ __forceinline__ float gate(const bsg_rows& x, int dtype, int e, int t, int h) {
  return dtype == BSG_BF16 ? (float)*row<bf16>(x, e, t, h) : *row<float>(x, e, t, h);
}
__device__ __forceinline__ void gate_out(const bsg_rows& x, int dtype, int e, int t, int h, float v) {
  if (dtype == BSG_BF16) *row_out<bf16>(x, e, t, h) = (bf16)v;
  else *row_out<float>(x, e, t, h) = v;
}
__device__ __forceinline__ int steps_of(const bsg_delta& a, int e) {
  return a.lengths ? min(max(a.lengths[e], 0), a.steps) : a.steps;
}

// The gates of a chunk, one lane of a wave per step.
struct Gates {
  float hi[C], lo[C];              // c_i
  float in[C], out[C], beta[C];
  int episode[C];                  // episodes begun in the chunk up to i
  float across;
};
__device__ __forceinline__ void read_gates(Gates& s, const bsg_delta& a, int e, int h, int t0, int rows, int lane) {
  const bool on = lane < rows;
  double c = on ? (double)fmaxf(gate(a.g, a.gate_dtype, e, t0 + lane, h), LOWEST) : 0.0;
  const bool f = on && a.first && a.first[e * a.first_env + (t0 + lane) * a.first_step] != 0;
  const unsigned long long begun = __ballot(f);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_up(c, d);
    if (lane >= d) c += o;
  }
  const double last = __shfl(c, 63);
  const int ep = __popcll(begun & (~0ull >> (63 - lane))), all = __popcll(begun);
  s.hi[lane] = (float)c;
  s.lo[lane] = (float)(c - (double)(float)c);
  s.in[lane] = ep == 0 ? expf((float)c) : 0.0f;
  s.out[lane] = ep == all ? expf((float)(last - c)) : 0.0f;
  s.beta[lane] = on ? gate(a.beta, a.gate_dtype, e, t0 + lane, h) : 0.0f;
  s.episode[lane] = ep;
  if (lane == 0) s.across = all == 0 ? expf((float)last) : 0.0f;
}
__device__ __forceinline__ float decay(const Gates& s, int i, int j) {
  return s.episode[i] == s.episode[j] ? expf((s.hi[i] - s.hi[j]) + (s.lo[i] - s.lo[j])) : 0.0f;
}

// What the passes along a rollout share of a chunk.  A workgroup of NW waves handles one env and
// value head; wave w owns the 16 value columns 16 w .. 16 w + 15 and keeps their part of the state
// in registers (as D tiles, whose rows are the key dimension), so the waves only meet over the
// C x C matrices.
template <class T, int DK>
struct Chunk {
  T k[C * pitch<T>(DK)], q[C * pitch<T>(DK)];
  float n[C * AP];                 // minus the matrix of the system, below the diagonal
  float p[C * AP];                 // P, its diagonal blocks filled with zeros above
  float inv[4 * 16 * IP];          // inverses of the system's diagonal blocks
  Gates gates;
};

// N and P, then the inverses.  BACK: the system is (I + diag(beta) N)^T, else I + N diag(beta).
template <class T, int DK, int NW, bool BACK>
__device__ __forceinline__ void solve_chunk(Chunk<T, DK>& s, float scale, int lane, int w) {
  constexpr int LD = pitch<T>(DK);
  const int m = lane & 15, g = lane >> 4;
  // eight strips of 16 rows, N's in rising and P's in falling length, over the waves
  for (int task = w; task < 8; task += NW) {
    const bool isP = task >= 4;
    const int b = isP ? 7 - task : task;
    const T* rows = (isP ? s.q : s.k) + (16 * b + m) * LD;
    Frag<T> af[DK / 32];
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) af[c] = load_run(rows, 32 * c, g);
    for (int u = 0; u <= b; ++u) {
      f32x4 d = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < DK / 32; ++c) mma(d, af[c], load_run(s.k + (16 * u + m) * LD, 32 * c, g));
      const int j = 16 * u + m;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * b + 4 * g + r;
        const float f = decay(s.gates, i, j);
        if (isP) s.p[i * AP + j] = j <= i ? scale * f * d[r] : 0.0f;
        else s.n[i * AP + j] = j < i ? -s.gates.beta[BACK ? i : j] * f * d[r] : 0.0f;
      }
    }
  }
  __syncthreads();
  if (w == 0) {                    // lane: block g, column m, by substitution down the rows
    float x[16];
    const float* nb = s.n + 16 * g * AP + 16 * g;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = i == m ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) x[i] = fmaf(nb[i * AP + j], x[j], x[i]);
      s.inv[(16 * g + i) * IP + m] = x[i];
    }
  }
}

// ---- forward -------------------------------------------------------------------------------
template <class T, int DK, int NW>
__global__ __launch_bounds__(64 * NW) void forward_kernel(bsg_delta a) {
  constexpr int LD = pitch<T>(DK), DT = DK / 16, DV = 16 * NW;
  __shared__ __align__(16) Chunk<T, DK> s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % a.heads_v, e = blockIdx.x / a.heads_v, hk = h / (a.heads_v / a.heads_k);
  const int n = steps_of(a, e), col = 16 * w + m;
  const int chunks = (a.steps + C - 1) / C;
  const int64_t eh = (int64_t)e * a.heads_v + h;

  f32x4 S[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[d][r] = a.state ? a.state[(eh * DK + 16 * d + 4 * g + r) * DV + col] : 0.0f;

  for (int ch = 0; ch < chunks; ++ch) {
    const int t0 = ch * C, rows = min(C, n - t0);
    if (rows <= 0) {               // padding: zeros
      for (int i = tid; i < min(C, a.steps - t0) * DV; i += 64 * NW) row_out<T>(a.out, e, t0 + i / DV, h)[i % DV] = (T)0.0f;
      continue;
    }
    f32x4 v[4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * b + 4 * g + r;
        v[b][r] = t < rows ? (float)row<T>(a.v, e, t0 + t, h)[col] : 0.0f;
      }
    __syncthreads();
    stage<T, DK, C>(s.k, row<T>(a.k, e, t0, hk), a.k.step, rows, tid, 64 * NW);
    stage<T, DK, C>(s.q, row<T>(a.q, e, t0, hk), a.q.step, rows, tid, 64 * NW);
    if (w == 0) read_gates(s.gates, a, e, h, t0, rows, lane);
    __syncthreads();
    solve_chunk<T, DK, NW, false>(s, a.scale, lane, w);

    if (a.kept_states) {
      float* ks = a.kept_states + (eh * chunks + ch) * DK * DV + col;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) ks[(16 * d + 4 * g + r) * DV] = S[d][r];
    }
    // K S and Q S
    f32x4 x[4], o[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] = o[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      WideOf<T, 3> sw;
      split(sw, join(S[2 * c], S[2 * c + 1]));
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        mma<T>(x[b], load_tile(s.k + (16 * b + m) * LD, 32 * c, g), sw);
        mma<T>(o[b], load_tile(s.q + (16 * b + m) * LD, 32 * c, g), sw);
      }
    }
    f32x4 beta[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 in = *reinterpret_cast<const f32x4*>(&s.gates.in[16 * b + 4 * g]);
      beta[b] = *reinterpret_cast<const f32x4*>(&s.gates.beta[16 * b + 4 * g]);
      x[b] = v[b] - in * x[b];
      o[b] *= in * a.scale;
    }
    __syncthreads();               // the inverses are there
    f32x4 W[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int u = 0; u < b; ++u)
        mma16(x[b], *reinterpret_cast<const f32x4*>(&s.n[(16 * b + m) * AP + 16 * u + 4 * g]), W[u]);
      W[b] = f32x4{0, 0, 0, 0};
      mma16(W[b], *reinterpret_cast<const f32x4*>(&s.inv[(16 * b + m) * IP + 4 * g]), x[b]);
    }
    if (a.kept_w) {
      float* kw = a.kept_w + (eh * chunks + ch) * C * DV + col;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) kw[(16 * b + 4 * g + r) * DV] = W[b][r];
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) W[b] *= beta[b];       // U
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int u = 0; u <= b; ++u)
        mma16(o[b], *reinterpret_cast<const f32x4*>(&s.p[(16 * b + m) * AP + 16 * u + 4 * g]), W[u]);
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * b + 4 * g + r;
        if (t0 + t < a.steps) row_out<T>(a.out, e, t0 + t, h)[col] = (T)(t < rows ? o[b][r] : 0.0f);
      }
#pragma unroll
    for (int d = 0; d < DT; ++d) S[d] *= s.gates.across;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f32x4 u[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) u[i] = W[2 * c + i] * *reinterpret_cast<const f32x4*>(&s.gates.out[16 * (2 * c + i) + 4 * g]);
      WideOf<T, 3> uw;
      split(uw, join(u[0], u[1]));
#pragma unroll
      for (int d = 0; d < DT; ++d) mma<T>(S[d], load_col(s.k, LD, 32 * c, 16 * d, lane), uw);
    }
  }
  if (a.final_state) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.final_state[(eh * DK + 16 * d + 4 * g + r) * DV + col] = S[d][r];
  }
}

// ---- backward along the rollout ------------------------------------------------------------
// The gradient of the state, from the last chunk to the first, and with it M and v'.  Every
// product's columns are value columns, so a wave works on its 16 alone, as in the forward pass.
template <class T, int DK, int NW>
__global__ __launch_bounds__(64 * NW) void backward_state_kernel(bsg_delta a) {
  constexpr int LD = pitch<T>(DK), DT = DK / 16, DV = 16 * NW;
  __shared__ __align__(16) Chunk<T, DK> s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int h = blockIdx.x % a.heads_v, e = blockIdx.x / a.heads_v, hk = h / (a.heads_v / a.heads_k);
  const int n = steps_of(a, e), col = 16 * w + m;
  const int chunks = (a.steps + C - 1) / C;
  const int64_t eh = (int64_t)e * a.heads_v + h;

  f32x4 D[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      D[d][r] = a.dfinal ? a.dfinal[(eh * DK + 16 * d + 4 * g + r) * DV + col] : 0.0f;

  for (int ch = chunks - 1; ch >= 0; --ch) {
    const int t0 = ch * C, rows = min(C, n - t0);
    if (rows <= 0) {
      for (int i = tid; i < min(C, a.steps - t0) * DV; i += 64 * NW) row_out<T>(a.dv, e, t0 + i / DV, h)[i % DV] = (T)0.0f;
      continue;
    }
    f32x4 go[4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * b + 4 * g + r;
        go[b][r] = t < rows ? (float)row<T>(a.dout, e, t0 + t, h)[col] : 0.0f;
      }
    __syncthreads();
    stage<T, DK, C>(s.k, row<T>(a.k, e, t0, hk), a.k.step, rows, tid, 64 * NW);
    stage<T, DK, C>(s.q, row<T>(a.q, e, t0, hk), a.q.step, rows, tid, 64 * NW);
    if (w == 0) read_gates(s.gates, a, e, h, t0, rows, lane);
    __syncthreads();
    solve_chunk<T, DK, NW, true>(s, a.scale, lane, w);

    float* ws = a.work_states + (eh * chunks + ch) * DK * DV + col;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) ws[(16 * d + 4 * g + r) * DV] = D[d][r];

    f32x4 x[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      WideOf<T, 3> dw;
      split(dw, join(D[2 * c], D[2 * c + 1]));
#pragma unroll
      for (int b = 0; b < 4; ++b) mma<T>(x[b], load_tile(s.k + (16 * b + m) * LD, 32 * c, g), dw);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      x[b] *= *reinterpret_cast<const f32x4*>(&s.gates.out[16 * b + 4 * g]);
#pragma unroll
      for (int u = b; u < 4; ++u) {
        const float* p = &s.p[(16 * u + 4 * g) * AP + 16 * b + m];
        mma16(x[b], f32x4{p[0], p[AP], p[2 * AP], p[3 * AP]}, go[u]);
      }
    }
    __syncthreads();               // the inverses are there
    f32x4 M[4];
#pragma unroll
    for (int b = 3; b >= 0; --b) {
#pragma unroll
      for (int u = b + 1; u < 4; ++u) {
        const float* p = &s.n[(16 * u + 4 * g) * AP + 16 * b + m];
        mma16(x[b], f32x4{p[0], p[AP], p[2 * AP], p[3 * AP]}, M[u]);
      }
      const float* p = &s.inv[(16 * b + 4 * g) * IP + m];
      M[b] = f32x4{0, 0, 0, 0};
      mma16(M[b], f32x4{p[0], p[IP], p[2 * IP], p[3 * IP]}, x[b]);
    }
    float* wm = a.work_w + (eh * chunks + ch) * C * DV + col;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 beta = *reinterpret_cast<const f32x4*>(&s.gates.beta[16 * b + 4 * g]);
      const f32x4 in = *reinterpret_cast<const f32x4*>(&s.gates.in[16 * b + 4 * g]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * b + 4 * g + r;
        wm[t * DV] = M[b][r];
        if (t0 + t < a.steps) row_out<T>(a.dv, e, t0 + t, h)[col] = (T)(t < rows ? beta[r] * M[b][r] : 0.0f);
      }
      M[b] *= beta * in * -1.0f;
      go[b] *= in * a.scale;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) D[d] *= s.gates.across;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      WideOf<T, 3> lw, ow;
      split(lw, join(M[2 * c], M[2 * c + 1]));
      split(ow, join(go[2 * c], go[2 * c + 1]));
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        mma<T>(D[d], load_col(s.k, LD, 32 * c, 16 * d, lane), lw);
        mma<T>(D[d], load_col(s.q, LD, 32 * c, 16 * d, lane), ow);
      }
    }
  }
  if (a.dstate) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.dstate[(eh * DK + 16 * d + 4 * g + r) * DV + col] = D[d][r];
  }
}

// ---- backward inside the chunks ------------------------------------------------------------
// q', k', beta', g' of one chunk, env and key head, all chunks side by side: a wave owns 16 steps.
// The matrices o'.w and m.w are needed by rows (for q', kr') and by columns (for kw'); both are
// computed, each in the layout in which it is the B operand of what follows, which costs less than
// a turn through LDS.  The value dimension is walked in slices of 32, the value heads that share
// the key head one after the other, their q' and k' added up in registers.
constexpr int SL = 32;
template <class T, int R>
struct WideRows {                  // an R x SL tile of fp32 values as operand parts of type T
  static constexpr int n = Parts<T, 2>::n, LD = pitch<T>(SL);
  T p[n][R * LD];
  __device__ __forceinline__ void put(int r, int c, const f32x4& x) {
    f32x4 rest = x;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      store4(&p[i][r * LD + c], rest);
      if (i + 1 < n) rest -= widen(*reinterpret_cast<const Half<T>*>(&p[i][r * LD + c]));
    }
  }
  __device__ __forceinline__ Wide<T, n> get(int r, int g) const {
    Wide<T, n> w;
#pragma unroll
    for (int i = 0; i < n; ++i) w.p[i] = load_run(&p[i][r * LD], 0, g);
    return w;
  }
};
template <class T, int N> __device__ __forceinline__ f32x8 whole(const Wide<T, N>& w) {
  f32x8 x = widen(w.p[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) x += widen(w.p[i]);
  return x;
}

template <class T, int DK>
struct Inside {
  T k[C * pitch<T>(DK)], q[C * pitch<T>(DK)], go[C * pitch<T>(SL)];
  WideRows<T, C> w, mu;
  WideRows<T, DK> st, ds;
  Gates gates;
  float dc[C], part[8];
};

template <class T, int DK>
__global__ __launch_bounds__(256) void backward_chunk_kernel(bsg_delta a) {
  constexpr int LD = pitch<T>(DK), DT = DK / 16, GL = pitch<T>(SL);
  __shared__ __align__(16) Inside<T, DK> s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int chunks = (a.steps + C - 1) / C, group = a.heads_v / a.heads_k, DV = a.dim_v;
  const int ch = blockIdx.x % chunks, ehk = blockIdx.x / chunks, hk = ehk % a.heads_k, e = ehk / a.heads_k;
  const int n = steps_of(a, e), t0 = ch * C, rows = min(C, n - t0), all = min(C, a.steps - t0);
  const int own = 16 * w + m;
  if (rows <= 0) {
    for (int i = tid; i < all * DK; i += 256) {
      row_out<T>(a.dq, e, t0 + i / DK, hk)[i % DK] = (T)0.0f;
      row_out<T>(a.dk, e, t0 + i / DK, hk)[i % DK] = (T)0.0f;
    }
    for (int i = tid; i < all * group; i += 256) {
      gate_out(a.dg, a.gate_dtype, e, t0 + i / group, hk * group + i % group, 0.0f);
      gate_out(a.dbeta, a.gate_dtype, e, t0 + i / group, hk * group + i % group, 0.0f);
    }
    return;
  }
  stage<T, DK, C>(s.k, row<T>(a.k, e, t0, hk), a.k.step, rows, tid, 256);
  stage<T, DK, C>(s.q, row<T>(a.q, e, t0, hk), a.q.step, rows, tid, 256);
  f32x4 dq[DT], dk[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) dq[d] = dk[d] = f32x4{0, 0, 0, 0};

  for (int h = hk * group; h < (hk + 1) * group; ++h) {
    const int64_t ehc = ((int64_t)e * a.heads_v + h) * chunks + ch;
    f32x4 OWt[4], MWt[4], OW[4], MW[4], X1[DT], X2[DT], X3[DT];
#pragma unroll
    for (int b = 0; b < 4; ++b) OWt[b] = MWt[b] = OW[b] = MW[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < DT; ++d) X1[d] = X2[d] = X3[d] = f32x4{0, 0, 0, 0};
    float dbeta = 0.0f, sd = 0.0f;
    for (int v0 = 0; v0 < DV; v0 += SL) {
      __syncthreads();
      if (v0 == 0 && w == 0) read_gates(s.gates, a, e, h, t0, rows, lane);
      stage<T, SL, C>(s.go, row<T>(a.dout, e, t0, h) + v0, a.dout.step, rows, tid, 256);
      for (int i = tid; i < C * SL / 4; i += 256) {
        const int r = i / (SL / 4), c = i % (SL / 4) * 4;
        const int64_t at = (ehc * C + r) * DV + v0 + c;
        s.w.put(r, c, *reinterpret_cast<const f32x4*>(a.kept_w + at));
        s.mu.put(r, c, *reinterpret_cast<const f32x4*>(a.work_w + at));
      }
      for (int i = tid; i < DK * SL / 4; i += 256) {
        const int r = i / (SL / 4), c = i % (SL / 4) * 4;
        const int64_t at = (ehc * DK + r) * DV + v0 + c;
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.kept_states + at);
        const f32x4 y = *reinterpret_cast<const f32x4*>(a.work_states + at);
        s.st.put(r, c, x);
        s.ds.put(r, c, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) sd = fmaf(x[j], y[j], sd);
      }
      __syncthreads();
      const Frag<T> go = load_run(s.go + own * GL, 0, g);
      const WideOf<T, 2> wf = s.w.get(own, g), mf = s.mu.get(own, g);
      const f32x8 wx = whole(wf), mx = whole(mf);
#pragma unroll
      for (int j = 0; j < 8; ++j) dbeta = fmaf(wx[j], mx[j], dbeta);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (b <= w) {
          const WideOf<T, 2> x = s.w.get(16 * b + m, g);
          mma<T>(OWt[b], x, go);
          mma<T>(MWt[b], x, mf);
        }
        if (b >= w) {
          mma<T>(OW[b], load_run(s.go + (16 * b + m) * GL, 0, g), wf);
          mma<T>(MW[b], s.mu.get(16 * b + m, g), wf);
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const WideOf<T, 2> x = s.st.get(16 * d + m, g), y = s.ds.get(16 * d + m, g);
        mma<T>(X1[d], x, go);
        mma<T>(X2[d], x, mf);
        mma<T>(X3[d], y, wf);
      }
    }
    // scale by the gates of the wave's own step (its lane) and add the chunk's own terms
    const Gates& G = s.gates;
    const float bi = G.beta[own], in = G.in[own], out = G.out[own];
    float y = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 k = widen(*reinterpret_cast<const Half<T>*>(&s.k[own * LD + 16 * d + 4 * g]));
      X1[d] *= a.scale * in;
      X2[d] *= -bi * in;
      X3[d] *= out * bi;
#pragma unroll
      for (int r = 0; r < 4; ++r) y = fmaf(k[r], X3[d][r], y);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (2 * c <= w) {            // rows j of tiles 2c, 2c + 1 against the own step i
        f32x4 f1[2], f2[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * (2 * c + u) + 4 * g + r;
            const float f = j <= own ? decay(G, own, j) * G.beta[j] : 0.0f;
            f1[u][r] = a.scale * f * OWt[2 * c + u][r];
            f2[u][r] = j < own ? -bi * f * MWt[2 * c + u][r] : 0.0f;
          }
        WideOf<T, 2> w1, w2;
        split(w1, join(f1[0], f1[1]));
        split(w2, join(f2[0], f2[1]));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const Frag<T> k = load_col(s.k, LD, 32 * c, 16 * d, lane);
          mma<T>(X1[d], k, w1);
          mma<T>(X2[d], k, w2);
        }
      }
      if (2 * c + 1 >= w) {        // rows i of tiles 2c, 2c + 1 against the own step j
        f32x4 f1[2], f2[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 16 * (2 * c + u) + 4 * g + r;
            const float f = i >= own ? decay(G, i, own) * bi : 0.0f;
            f1[u][r] = a.scale * f * OW[2 * c + u][r];
            f2[u][r] = i > own ? -G.beta[i] * f * MW[2 * c + u][r] : 0.0f;
          }
        WideOf<T, 2> w1, w2;
        split(w1, join(f1[0], f1[1]));
        split(w2, join(f2[0], f2[1]));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          mma<T>(X3[d], load_col(s.q, LD, 32 * c, 16 * d, lane), w1);
          mma<T>(X3[d], load_col(s.k, LD, 32 * c, 16 * d, lane), w2);
        }
      }
    }
    float dc = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 k = widen(*reinterpret_cast<const Half<T>*>(&s.k[own * LD + 16 * d + 4 * g]));
      const f32x4 q = widen(*reinterpret_cast<const Half<T>*>(&s.q[own * LD + 16 * d + 4 * g]));
#pragma unroll
      for (int r = 0; r < 4; ++r) dc = fmaf(q[r], X1[d][r], fmaf(k[r], X2[d][r] - X3[d][r], dc));
      dq[d] += X1[d];
      dk[d] += X2[d] + X3[d];
    }
    dc = sum_groups(dc);
    dbeta = sum_groups(dbeta);
    // the chunk's last step: across <S, D> + sum_j k_j.(out_j D u_j)
    y += G.across * sd;
#pragma unroll
    for (int d = 32; d >= 1; d /= 2) y += __shfl_xor(y, d);
    if (g == 0) s.dc[own] = dc;
    if (lane == 0) s.part[w] = y;
    if (g == 0 && t0 + own < a.steps)
      gate_out(a.dbeta, a.gate_dtype, e, t0 + own, h, own < rows ? dbeta : 0.0f);
    __syncthreads();
    if (w == 0) {
      float x = s.dc[lane];
      if (lane == 63) x += (s.part[0] + s.part[1]) + (s.part[2] + s.part[3]);
      const int ep = G.episode[lane], before = lane ? G.episode[lane - 1] : 0;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const float o = __shfl_down(x, d);
        const int oe = __shfl_down(ep, d);
        if (lane + d < 64 && oe == ep) x += o;
      }
      // a first step's decay meets no state
      if (t0 + lane < a.steps)
        gate_out(a.dg, a.gate_dtype, e, t0 + lane, h, lane < rows && ep == before ? x : 0.0f);
    }
  }
  if (t0 + own >= a.steps) return;
  T *oq = row_out<T>(a.dq, e, t0 + own, hk), *ok = row_out<T>(a.dk, e, t0 + own, hk);
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    store4(oq + 16 * d + 4 * g, own < rows ? dq[d] : f32x4{0, 0, 0, 0});
    store4(ok + 16 * d + 4 * g, own < rows ? dk[d] : f32x4{0, 0, 0, 0});
  }
}

// ---- acting --------------------------------------------------------------------------------
// One wave per env, value head and slice of value columns: the slice of the state in registers,
// both sums over it (S^T k and S^T q) in one pass, then the update.  Lanes hold four columns;
// S'^T q = (S + k u^T)^T q = S^T q + (k.q) u.
template <class T, int DK, int DV>
__global__ __launch_bounds__(256) void step_kernel(bsg_delta a, int64_t waves) {
  constexpr int COLS = DV == 32 || DK == 128 ? 32 : 64, L = COLS / 4, RG = 64 / L, N = DK / RG, SLICES = DV / COLS;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= waves) return;
  const int lane = threadIdx.x & 63, rg = lane / L;
  const int64_t eh = id / SLICES;
  const int c0 = (int)(id % SLICES) * COLS + lane % L * 4;
  const int h = (int)(eh % a.heads_v), e = (int)(eh / a.heads_v), hk = h / (a.heads_v / a.heads_k);
  const bool first = a.first && a.first[e * a.first_env] != 0;
  float* st = a.final_state + eh * DK * DV + c0;
  f32x4 S[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    S[i] = first ? f32x4{0, 0, 0, 0} : *reinterpret_cast<const f32x4*>(st + (i * RG + rg) * DV);
  const T *kr = row<T>(a.k, e, 0, hk), *qr = row<T>(a.q, e, 0, hk);
  const f32x4 v = widen(*reinterpret_cast<const Half<T>*>(row<T>(a.v, e, 0, h) + c0));
  const float alpha = expf(fmaxf(gate(a.g, a.gate_dtype, e, 0, h), LOWEST)), beta = gate(a.beta, a.gate_dtype, e, 0, h);
  float k[N], kq = 0.0f;
  f32x4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    k[i] = (float)kr[i * RG + rg];
    const float q = (float)qr[i * RG + rg];
    S[i] *= alpha;
    kq = fmaf(k[i], q, kq);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sk[j] = fmaf(k[i], S[i][j], sk[j]);
      sq[j] = fmaf(q, S[i][j], sq[j]);
    }
  }
#pragma unroll
  for (int d = L; d < 64; d *= 2) {
    kq += __shfl_xor(kq, d);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sk[j] += __shfl_xor(sk[j], d);
      sq[j] += __shfl_xor(sq[j], d);
    }
  }
  const f32x4 u = (v - sk) * beta;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) S[i][j] = fmaf(k[i], u[j], S[i][j]);
    *reinterpret_cast<f32x4*>(st + (i * RG + rg) * DV) = S[i];
  }
  if (rg == 0) store4(row_out<T>(a.out, e, 0, h) + c0, (sq + u * kq) * a.scale);
}

enum { FORWARD, BACKWARD, STEP };

template <class T, int DK, int NW>
hipError_t run(const bsg_delta& a, int what, hipStream_t st) {
  const unsigned rows = (unsigned)(a.num_envs * a.heads_v);
  if (what == STEP) {
    constexpr int DV = 16 * NW, slices = DV / (DV == 32 || DK == 128 ? 32 : 64);
    const int64_t waves = (int64_t)rows * slices;
    step_kernel<T, DK, DV><<<dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st>>>(a, waves);
  } else if (what == FORWARD) {
    forward_kernel<T, DK, NW><<<dim3(rows), dim3(64 * NW), 0, st>>>(a);
  } else {
    backward_state_kernel<T, DK, NW><<<dim3(rows), dim3(64 * NW), 0, st>>>(a);
    const int chunks = (a.steps + C - 1) / C;
    backward_chunk_kernel<T, DK><<<dim3((unsigned)(a.num_envs * a.heads_k * chunks)), dim3(256), 0, st>>>(a);
  }
  return hipGetLastError();
}
template <class T, int DK>
hipError_t run(const bsg_delta& a, int what, hipStream_t st) {
  return a.dim_v == 32 ? run<T, DK, 2>(a, what, st) : a.dim_v == 64 ? run<T, DK, 4>(a, what, st) : run<T, DK, 8>(a, what, st);
}
template <class T>
hipError_t run(const bsg_delta& a, int what, hipStream_t st) {
  return a.dim_k == 32 ? run<T, 32>(a, what, st) : a.dim_k == 64 ? run<T, 64>(a, what, st) : run<T, 128>(a, what, st);
}
hipError_t run(const bsg_delta& a, int what, hipStream_t st) {
  return a.dtype == BSG_BF16 ? run<bf16>(a, what, st) : run<float>(a, what, st);
}

}  // namespace

namespace bsg {

// Shapes, strides and pointers are validated by the bsg_delta_* entry points (bsg_abi.cpp).
hipError_t launch_delta_forward(const bsg_delta& a, hipStream_t st) { return run(a, FORWARD, st); }
hipError_t launch_delta_backward(const bsg_delta& a, hipStream_t st) { return run(a, BACKWARD, st); }
hipError_t launch_delta_step(const bsg_delta& a, hipStream_t st) { return run(a, STEP, st); }

}  // namespace bsg
