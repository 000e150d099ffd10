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
constexpr int IP = 20;             // row pitch of a 16 x 16 tile of fp32 in LDS
constexpr float LOWEST = -1e5f;    // the least log decay: its exponential is 0
__device__ __forceinline__ float at_least_lowest(float g) { return g < LOWEST ? LOWEST : g; }   // NaN stays

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

// The gates of a chunk, one lane of a wave per step.  c is kept in units of log 2 (v_exp_f32 is a
// power of two, and the product with log2 e is rounded in double).
struct Gates {
  float hi[C], lo[C];              // c_i
  float in[C], out[C], beta[C];
  int episode[C];                  // episodes begun in the chunk up to i
  float across, pad[3];
};
// The kernel's arguments, read anew: what is needed once a chunk or once a head is then not kept in
// scalar registers all along (the compiler takes the address for a new one each time).
__device__ __forceinline__ const bsg_delta& arguments() {
  typedef const __attribute__((address_space(4))) bsg_delta* Args;
  Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const bsg_delta*)p;
}

// An env's and head's rows along the steps.
template <class T> struct Steps {
  T* p;
  int64_t step;
  __device__ __forceinline__ T* at(int t) const { return p + t * step; }
};
template <class T> __device__ __forceinline__ Steps<T> steps_in(const bsg_rows& x, int e, int h, int col = 0) {
  return {static_cast<T*>(x.p) + e * x.env + h * x.head + col, x.step};
}
struct GateSteps {
  const char *g, *beta;
  const uint8_t* first;
  int64_t g_step, beta_step, first_step;   // in bytes
  bool half;
  __device__ __forceinline__ GateSteps(const bsg_delta& a, int e, int h) {
    half = a.gate_dtype == BSG_BF16;
    const int b = half ? 2 : 4;
    g = static_cast<const char*>(a.g.p) + (e * a.g.env + h * a.g.head) * b;
    beta = static_cast<const char*>(a.beta.p) + (e * a.beta.env + h * a.beta.head) * b;
    first = a.first ? a.first + e * a.first_env : nullptr;
    g_step = a.g.step * b, beta_step = a.beta.step * b, first_step = a.first_step;
  }
};
// A lane's step as it lies in memory, not looked at before make_gates (the loads stay in flight).
struct RawGates { uint32_t g, beta, first; };
__device__ __forceinline__ RawGates load_gates(const GateSteps& s, int t0, int rows, int lane) {
  RawGates r = {0, 0, 0};
  if (lane < rows) {
    const int t = t0 + lane;
    if (s.half) {
      r.g = *reinterpret_cast<const uint16_t*>(s.g + t * s.g_step);
      r.beta = *reinterpret_cast<const uint16_t*>(s.beta + t * s.beta_step);
    } else {
      r.g = *reinterpret_cast<const uint32_t*>(s.g + t * s.g_step);
      r.beta = *reinterpret_cast<const uint32_t*>(s.beta + t * s.beta_step);
    }
    if (s.first) r.first = s.first[t * s.first_step];
  }
  return r;
}
__device__ __forceinline__ void make_gates(Gates& s, const RawGates& raw, bool half, int lane) {
  asm volatile("" : "+v"(lane));   // else a comparison's mask a step stays in scalar registers all along
  double c = (double)at_least_lowest(__uint_as_float(half ? raw.g << 16 : raw.g)) * 1.4426950408889634074;
  const unsigned long long begun = __ballot(raw.first != 0);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_up(c, d);
    if (lane >= d) c += o;
  }
  const double last = __shfl(c, 63);
  const int ep = __popcll(begun & (~0ull >> (63 - lane))), all = __popcll(begun);
  s.hi[lane] = (float)c;
  s.lo[lane] = (float)(c - (double)(float)c);
  s.in[lane] = ep == 0 ? __builtin_amdgcn_exp2f((float)c) : 0.0f;
  s.out[lane] = ep == all ? __builtin_amdgcn_exp2f((float)(last - c)) : 0.0f;
  s.beta[lane] = __uint_as_float(half ? raw.beta << 16 : raw.beta);
  s.episode[lane] = ep;
  if (lane == 0) s.across = all == 0 ? __builtin_amdgcn_exp2f((float)last) : 0.0f;
}
// G_ij of four rows i = row..row + 3 and the step j (FROM: of the rows j and the step i), for i >= j;
// no branch: another episode's exponent is lowered until nothing is left.
struct Step { float hi, lo; int episode; };
__device__ __forceinline__ Step step_of(const Gates& s, int i) { return {s.hi[i], s.lo[i], s.episode[i]}; }
template <bool FROM>
__device__ __forceinline__ f32x4 decays(const Gates& s, int row, const Step& o) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const f32x4 hi = *reinterpret_cast<const f32x4*>(&s.hi[row]), lo = *reinterpret_cast<const f32x4*>(&s.lo[row]);
  const i32x4 ep = *reinterpret_cast<const i32x4*>(&s.episode[row]);
  f32x4 f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float x = FROM ? (o.hi - hi[r]) + (o.lo - lo[r]) : (hi[r] - o.hi) + (lo[r] - o.lo);
    f[r] = __builtin_amdgcn_exp2f(ep[r] == o.episode ? x : -1e9f);
  }
  return f;
}

// The passes along a rollout.  ALONE solves each chunk where it needs it.  Where the chunks are solved
// beforehand, CARRY takes each segment of the rollout to its transition and JOINED runs all segments side
// by side, each from the state that the joined transitions give it.
enum Pass { ALONE, JOINED, CARRY };

// What the passes along a rollout need of a chunk besides its rows (ALL: with P; HERE: solved in place).
template <class T, bool ALL, bool HERE>
struct Solved {
  static constexpr int PD = pitch<T>(C), parts = Parts<T, 2>::n;
  T p[ALL ? parts : 1][ALL ? C * PD : Vec<T>::n];   // P in parts of type T, zeros above its diagonal
  float n[6 * 16 * IP];            // minus the matrix of the system: the tiles below the diagonal,
  float inv[4 * 16 * IP];          // ... the inverses of those on it,
  Gates gates[HERE ? 2 : 1];       // (of this chunk and the one that comes next)
  static constexpr int tile(int b, int u) { return (b * (b - 1) / 2 + u) * 16 * IP; }
  // ... and those themselves, needed for the inverses only, where P has zeros that no product reads: rows
  // 0..31, columns 32..63 (in LDS of their own: dims 32 at 600 x 300 544 against 515 us, dims 128 and 64 at
  // 300 x 300 833 against 777, where a workgroup more fits a CU).
  static constexpr int DP = PD * (int)sizeof(T) / 4;
  __device__ __forceinline__ float* diagonal(int b) {
    return reinterpret_cast<float*>(p[sizeof(T) == 2 ? b & 1 : 0] + (b >> 1) * 16 * PD + 32 + (sizeof(T) == 2 ? 0 : (b & 1) * 16));
  }
  __device__ __forceinline__ WideOf<T, 2> p_row(int r, int k0, int g) const {
    WideOf<T, 2> w;
#pragma unroll
    for (int i = 0; i < parts; ++i) w.p[i] = load_tile(&p[i][r * PD], k0, g);
    return w;
  }
  __device__ __forceinline__ WideOf<T, 2> p_col(int m0, int k0, int lane) const {
    WideOf<T, 2> w;
#pragma unroll
    for (int i = 0; i < parts; ++i) w.p[i] = load_col(p[i], PD, k0, m0, lane);
    return w;
  }
};
// ... which passes through memory up to the first gates where the chunks are solved beforehand.
template <class T> constexpr int solved_bytes() { return sizeof(Solved<T, true, false>); }
template <class T> constexpr int p_bytes() { return sizeof(Solved<T, true, false>::p); }

// A workgroup of NW waves handles 16 NW value columns of one env and value head; wave w owns 16 of
// them and keeps their part of the state in registers (as D tiles, whose rows are the key
// dimension), so the waves only meet over the C x C matrices.
template <class T, int DK, int NW, bool HERE = true, bool Q = true, bool V = sizeof(T) == 2>
struct Chunk {
  static constexpr int LD = pitch<T>(DK), VD = pitch<T>(16 * NW);
  T k[C * LD], q[Q ? C * LD : Vec<T>::n];
  T v[V ? C * VD : Vec<T>::n];       // v (dout), then, column by column, out (v')
  Solved<T, Q, HERE> s;
};
// Waves per SIMD that LDS leaves room for, two at most: what bounds the passes' registers.
template <class T, int DK, int NW> constexpr int waves_per_simd() {
  return NW == 2 ? 1 : NW == 8 || 2 * sizeof(Chunk<T, DK, NW>) <= 160 * 1024 ? 2 : 1;
}

// A wave's 16 columns of the value rows, as D tiles.  bf16 passes through LDS, so that memory sees 16
// bytes a lane, in and out; fp32, where 16 lanes make 64 bytes of a row, goes straight to and from
// registers, and the LDS that saves lets two workgroups share a CU.
template <class T, int NW, bool LDS>
struct Columns {
  static constexpr int NT = 64 * NW, VD = pitch<T>(16 * NW);
  Fetch<T, C, 16 * NW, NT> f;
  __device__ __forceinline__ void load(const T* p, int64_t stride, int rows, int tid, int) { f.load(p, stride, rows, tid); }
  __device__ __forceinline__ void store(T* s, int rows, int tid) { f.store(s, rows, tid); }
  __device__ __forceinline__ void get(f32x4 (&x)[4], const T* s, int, int w, int lane) const {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[b][r] = (float)s[(16 * b + 4 * (lane >> 4) + r) * VD + 16 * w + (lane & 15)];
  }
  // to LDS, and from there to memory; rows behind `rows` are padding: zeros, up to `all`
  static __device__ __forceinline__ void put(T* s, const f32x4 (&x)[4], T*, int64_t, int, int, int w, int lane) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[(16 * b + 4 * (lane >> 4) + r) * VD + 16 * w + (lane & 15)] = (T)x[b][r];
  }
  static __device__ __forceinline__ void write(const T* s, T* to, int64_t stride, int rows, int all, int w, int lane) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int V = Vec<T>::n, P = 16 / V;     // pieces to a row
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int r = (lane + 64 * i) / P, c = 16 * w + (lane + 64 * i) % P * V;
      u32x4 x = *reinterpret_cast<const u32x4*>(s + r * VD + c);
      if (r >= rows) x = u32x4{0, 0, 0, 0};
      if (r < all) *reinterpret_cast<u32x4*>(to + r * stride + c) = x;
    }
  }
};
template <class T, int NW>
struct Columns<T, NW, false> {
  f32x4 next[4], now[4];
  __device__ __forceinline__ void load(const T* p, int64_t stride, int rows, int tid, int col) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) next[b][r] = (float)p[min(16 * b + 4 * (tid % 64 >> 4) + r, rows - 1) * stride + col];
  }
  __device__ __forceinline__ void store(T*, int, int) {
#pragma unroll
    for (int b = 0; b < 4; ++b) now[b] = next[b];
  }
  __device__ __forceinline__ void get(f32x4 (&x)[4], const T*, int rows, int, int lane) const {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[b][r] = 16 * b + 4 * (lane >> 4) + r < rows ? now[b][r] : 0.0f;
  }
  static __device__ __forceinline__ void put(T*, const f32x4 (&x)[4], T* to, int64_t stride, int rows, int all, int w, int lane) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = 16 * b + 4 * (lane >> 4) + r;
        if (t < all) to[t * stride + 16 * w + (lane & 15)] = (T)(t < rows ? x[b][r] : 0.0f);
      }
  }
  static __device__ __forceinline__ void write(const T*, T*, int64_t, int, int, int, int) {}
};

// lane j of each row of 16 lanes, to all of them
template <int J> __device__ __forceinline__ float from_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + J, 0xf, 0xf, true));
}
// some columns x[c] of lane i's row: less n_iJ times row J of the inverse, which is done (and 0 before
// the column's own row)
template <int J, int N> __device__ __forceinline__ void eliminate(float (&x)[N], const float (&n)[16]) {
  if constexpr (J < 15) {
#pragma unroll
    for (int c = 0; c < N; ++c) x[c] = fmaf(from_lane<J>(x[c]), n[J], x[c]);
    eliminate<J + 1>(x, n);
  }
}

// The ten lower tiles of N and P (one decay serves both), then, after a barrier, the inverses: 16 / NW
// columns of each to a wave, a row to a lane; the substitution takes the rows before from their lanes
// (by one wave alone it held the others up: 102 against 89 us, 512x50 fp32).  The inverses are there after the caller's next barrier.
// BACK: the system is (I + diag(beta) N)^T, else I + N diag(beta).
template <class T, int DK, int NW, bool BACK, class X>
__device__ __forceinline__ void solve_chunk(X& x, const Gates& gates, float scale, int lane, int w) {
  constexpr int LD = pitch<T>(DK), PD = pitch<T>(C);
  asm volatile("" : "+v"(lane));
  auto& s = x.s;
  const int m = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t0 = 0; t0 < 10; t0 += NW) {
    const int t = min(t0 + w, 9);  // waves without one of their own repeat the last: no branch
    const int b = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3, u = t - b * (b + 1) / 2, j = 16 * u + m;
    f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      const Frag<T> kj = load_run(x.k + j * LD, 32 * c, g);
      mma(kk, load_run(x.k + (16 * b + m) * LD, 32 * c, g), kj);
      mma(qk, load_run(x.q + (16 * b + m) * LD, 32 * c, g), kj);
    }
    const float bj = gates.beta[j];
    const f32x4 bi = *reinterpret_cast<const f32x4*>(&gates.beta[16 * b + 4 * g]);
    const f32x4 f = decays<false>(gates, 16 * b + 4 * g, step_of(gates, j));
    const int np = b == u ? s.DP : IP;
    float* n = (b == u ? s.diagonal(b) : s.n + s.tile(b, u)) + 4 * g * np + m;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * b + 4 * g + r;
      n[r * np] = j < i ? -(BACK ? bi[r] : bj) * f[r] * kk[r] : 0.0f;
      float y = j <= i ? scale * f[r] * qk[r] : 0.0f;
#pragma unroll
      for (int o = 0; o < Parts<T, 2>::n; ++o) {
        const T z = (T)y;
        s.p[o][i * PD + j] = z;
        y -= (float)z;
      }
    }
  }
  __syncthreads();
  constexpr int N = 16 / NW;
  const int c0 = N * w;
  float v[N], n[16];               // lane: block g, row m
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(s.diagonal(g) + m * s.DP + j);
#pragma unroll
    for (int o = 0; o < 4; ++o) n[j + o] = y[o];
  }
#pragma unroll
  for (int c = 0; c < N; ++c) v[c] = c0 + c == m ? 1.0f : 0.0f;
  eliminate<0>(v, n);
#pragma unroll
  for (int c = 0; c < N; ++c) s.inv[(16 * g + m) * IP + c0 + c] = v[c];
}
// P's tiles above the diagonal that share a product step with one on it
template <class T>
__device__ __forceinline__ void clear_above(Solved<T, true, true>& s, int tid, int nt) {
  for (int i = tid; i < 2 * 256; i += nt) {
    const int b = i / 256 * 32, r = i % 256 / 16, c = i % 16;
#pragma unroll
    for (int o = 0; o < s.parts; ++o) s.p[o][(b + r) * s.PD + b + 16 + c] = (T)0.0f;
  }
}

// Few rows: the chunks are solved beforehand, all side by side, by workgroups of four waves.
template <class T, int DK, bool BACK>
__global__ __launch_bounds__(256) void solve_kernel(bsg_delta a) {
  __shared__ __align__(16) Chunk<T, DK, 4, true, true, false> s;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunks = (a.steps + C - 1) / C, ch = blockIdx.x % chunks, eh = blockIdx.x / chunks;
  const int h = eh % a.heads_v, e = eh / a.heads_v, hk = h / (a.heads_v / a.heads_k);
  const int t0 = ch * C, rows = min(C, steps_of(a, e) - t0);
  if (rows <= 0) return;
  Fetch<T, C, DK, 256> fk, fq;
  fk.load(row<T>(a.k, e, t0, hk), a.k.step, rows, tid);
  fq.load(row<T>(a.q, e, t0, hk), a.q.step, rows, tid);
  if (w == 0) {
    const GateSteps gate(a, e, h);
    make_gates(s.s.gates[0], load_gates(gate, t0, rows, lane), gate.half, lane);
  }
  clear_above(s.s, tid, 256);
  fk.store(s.k, rows, tid);
  fq.store(s.q, rows, tid);
  __syncthreads();
  solve_chunk<T, DK, 4, BACK>(s, s.s.gates[0], a.scale, lane, w);
  __syncthreads();
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  constexpr int N = solved_bytes<T>() / 16;
  u32x4* to = reinterpret_cast<u32x4*>(a.work) + ((int64_t)eh * chunks + ch) * N;
  const u32x4* from = reinterpret_cast<const u32x4*>(&s.s);
  for (int i = tid; i < N; i += 256) to[i] = from[i];
}
// ... and their results fetched a chunk ahead, as the rows are.
template <class T, int NT, bool ALL>
struct FetchSolved {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  static constexpr int skip = ALL ? 0 : p_bytes<T>() / 16, N = solved_bytes<T>() / 16 - skip, n = (N + NT - 1) / NT;
  u32x4 x[n];
  __device__ __forceinline__ void load(const void* work, int64_t chunk, int tid) {
    const u32x4* p = reinterpret_cast<const u32x4*>(work) + chunk * (N + skip) + skip;
#pragma unroll
    for (int i = 0; i < n; ++i) x[i] = p[min(tid + i * NT, N - 1)];
  }
  __device__ __forceinline__ void store(Solved<T, ALL, false>& s, int tid) const {
    u32x4* p = reinterpret_cast<u32x4*>(ALL ? (void*)&s : (void*)s.n);
#pragma unroll
    for (int i = 0; i < n; ++i)
      if (tid + i * NT < N) p[tid + i * NT] = x[i];
  }
};

// the first two parts: enough for what ends in an output of type T
__device__ __forceinline__ const Wide<float, 1>& front(const Wide<float, 1>& w) { return w; }
__device__ __forceinline__ Wide<bf16, 2> front(const Wide<bf16, 3>& w) { return Wide<bf16, 2>{{w.p[0], w.p[1]}}; }

// States and W (M) that only these kernels read lie as their D tiles do: 16 bytes a lane, wave by wave.
__device__ __forceinline__ float* tiles(float* p, int64_t chunk, int waves, int tiles_per_wave, int w, int lane) {
  return p + ((chunk * waves + w) * tiles_per_wave * 64 + lane) * 4;
}

// A rollout in segments of whole chunks.  What a segment does to the state before it is affine: with
// the products of its chunks' transitions A[dim_k][dim_k] (the pass run on the unit matrix, without
// values) and what it makes of no state, B[dim_k][dim_v], S' = A S + B.  `carry` holds, per row (env and
// value head) and boundary of segments, B by D tiles and A by the lanes that multiply it; join_kernel puts the state at the
// boundary in B's place.
struct Segments {
  float* carry;
  int count, chunks;               // segments to a rollout, chunks to a segment
};
__device__ __forceinline__ float* boundary(const Segments& seg, int64_t row, int at, int dk, int dv) {
  return seg.carry + (row * (seg.count - 1) + at) * dk * (dk + dv);
}

template <int DT>
__device__ __forceinline__ void put_carry(float* to, const f32x4 (&x)[DT], bool unit, int all, int c0, int w, int lane) {
  const int col = c0 + 16 * w + (lane & 15);
  if (!unit) {
    float* p = tiles(to, 0, 1, DT, c0 / 16 + w, lane);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(p + 256 * d) = x[d];
  } else if (col < 16 * DT) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        to[16 * DT * all + ((d * DT + col / 16) * 64 + col % 16 / 4 * 16 + 4 * (lane >> 4) + r) * 4 + col % 4] = x[d][r];
  }
}
// S' = A S + B from boundary to boundary (BACK: from the last one to the first).  A workgroup holds 16
// columns; a wave computes 16 rows of each product, and the waves meet in LDS after it.
template <int DK, bool BACK>
__global__ __launch_bounds__(4 * DK) void join_kernel(bsg_delta a, Segments seg) {
  constexpr int DT = DK / 16;
  __shared__ f32x4 sS[2][DT][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  const int all = a.dim_v, c0 = blockIdx.x % (all / 16) * 16, eh = blockIdx.x / (all / 16);
  const int live = (steps_of(a, eh / a.heads_v) + C - 1) / C;
  const int boundaries = (live + seg.chunks - 1) / seg.chunks - 1;
  if (boundaries <= 0) return;
  const float* start = BACK ? a.dfinal : a.state;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    sS[0][w][lane][r] = start ? start[((int64_t)eh * DK + 16 * w + 4 * g + r) * all + c0 + m] : 0.0f;
  struct Step {
    f32x4 a[DT], x;
  } even, odd;                     // of a boundary, loaded while the one before it is computed
  const auto at = [&](int i) { return boundary(seg, eh, BACK ? boundaries - 1 - i : i, DK, all); };
  const auto load = [&](Step& o, int i) {
    float* p = at(i);
    o.x = *reinterpret_cast<const f32x4*>(tiles(p, 0, 1, DT, c0 / 16, lane) + 256 * w);
#pragma unroll
    for (int u = 0; u < DT; ++u) o.a[u] = *reinterpret_cast<const f32x4*>(p + DK * all + ((w * DT + u) * 64 + lane) * 4);
  };
  const auto step = [&](Step& o, Step& next, int i) {
    load(next, min(i + 1, boundaries - 1));   // no branch: it would wait for all loads
    f32x4 y = {0, 0, 0, 0};        // two sums, so that products do not wait for each other
#pragma unroll
    for (int u = 0; u < DT; u += 2) {
      mma16(o.x, o.a[u], sS[i & 1][u][lane]);
      mma16(y, o.a[u + 1], sS[i & 1][u + 1][lane]);
    }
    o.x += y;
    *reinterpret_cast<f32x4*>(tiles(at(i), 0, 1, DT, c0 / 16, lane) + 256 * w) = o.x;
    sS[~i & 1][w][lane] = o.x;
    __syncthreads();
  };
  load(even, 0);
  __syncthreads();
  for (int i = 0; i < boundaries; i += 2) {
    step(even, odd, i);
    if (i + 1 < boundaries) step(odd, even, i + 1);
  }
}

// ---- forward -------------------------------------------------------------------------------
// Per chunk: X = V - in (K S), W by block substitution, O, S'.  K, Q, V come from memory a chunk ahead, the
// state stays in registers, and every product's columns are value columns, so that waves wait for each
// other only where the chunk is solved.  Measured: 512 envs x 300 steps, 4 heads, bf16, dim 64 198 us for
// 236 MB of rows and 336 MB of kept states and W (2.9 TB/s, 57 % of a large copy's rate); 512 x 50 fp32
// 90 us, half of it fp32 matrix instructions.  Two waves a SIMD (registers, LDS) do not cover their
// latencies: VALU 42 %, matrix cores 23 % busy.
template <class T, int DK, int NW, Pass PASS>
__global__ __launch_bounds__(64 * NW, (PASS == ALONE ? waves_per_simd<T, DK, NW>() : PASS == CARRY && sizeof(T) == 2 ? 2 : 1)) void forward_kernel(bsg_delta a, Segments seg) {
  constexpr int LD = pitch<T>(DK), DT = DK / 16, DV = 16 * NW, NT = 64 * NW;
  // rows a chunk ahead; not for fp32 solved in place (600 envs x 50 steps, dims 32: 186 -> 198 us)
  constexpr bool AHEAD = PASS != ALONE || sizeof(T) == 2;
  constexpr bool OUT = PASS != CARRY, LDS = sizeof(T) == 2;
  __shared__ __align__(16) Chunk<T, DK, NW, PASS == ALONE, OUT, LDS> s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  // the workgroup's columns of all (CARRY: and of the unit matrix's, behind them) and its segment
  const int all = PASS == ALONE ? DV : a.dim_v, groups = all / DV + (OUT ? 0 : (DK + DV - 1) / DV);
  const int segments = PASS == ALONE ? 1 : OUT ? seg.count : seg.count - 1, id = blockIdx.x / groups, part = id % segments;
  const int eh = id / segments, h = eh % a.heads_v, e = eh / a.heads_v, hk = h / (a.heads_v / a.heads_k);
  const bool unit = !OUT && (int)(blockIdx.x % groups) >= all / DV;
  const int c0 = (int)(blockIdx.x % groups) * DV - (unit ? all : 0), col = 16 * w + m;
  const int n = steps_of(a, e), chunks = (a.steps + C - 1) / C, live = (n + C - 1) / C;
  const int at = part;              // the segment
  const int begin = PASS == ALONE ? 0 : at * seg.chunks, end = PASS == ALONE ? live : min(begin + seg.chunks, live);
  if (!OUT && (part + 1) * seg.chunks >= live) return;   // no boundary before the rollout's end

  f32x4 S[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[d][r] = !OUT ? unit && 16 * d + 4 * g + r == c0 + col ? 1.0f : 0.0f
                     : at == 0 && a.state ? a.state[((int64_t)eh * DK + 16 * d + 4 * g + r) * all + c0 + col] : 0.0f;
  if (PASS == JOINED && at > 0 && begin < end) {
    const float* p = tiles(boundary(seg, eh, at - 1, DK, all), 0, 1, DT, c0 / 16 + w, lane);
#pragma unroll
    for (int d = 0; d < DT; ++d) S[d] = *reinterpret_cast<const f32x4*>(p + 256 * d);
  }

  Fetch<T, C, DK, NT> fk, fq;
  Columns<T, NW, LDS> fv;
  FetchSolved<T, NT, OUT> fs;
  RawGates raw = {0, 0, 0};
  const Steps<const T> k = steps_in<const T>(a.k, e, hk), q = steps_in<const T>(a.q, e, hk), v = steps_in<const T>(a.v, e, h, unit ? 0 : c0);
  const Steps<T> out = steps_in<T>(a.out, e, h, c0);
  const GateSteps gate(a, e, h);
  float *const ks = OUT && a.kept_states ? tiles(a.kept_states, (int64_t)eh * chunks, all / 16, DT, c0 / 16 + w, lane) : nullptr;
  float *const kw = OUT && a.kept_w ? tiles(a.kept_w, (int64_t)eh * chunks, all / 16, 4, c0 / 16 + w, lane) : nullptr;
  if (begin < end) {
    const int t0 = begin * C;
    if (AHEAD) {
      fk.load(k.at(t0), k.step, n - t0, tid);
      if (OUT) fq.load(q.at(t0), q.step, n - t0, tid);
      if (!unit) fv.load(v.at(t0), v.step, n - t0, tid, col);
    }
    if constexpr (PASS != ALONE) {
      fs.load(a.work, (int64_t)eh * chunks + begin, tid);
    } else {
      if (w == 0) make_gates(s.s.gates[0], load_gates(gate, 0, n, lane), gate.half, lane);
      clear_above(s.s, tid, NT);
    }
  }
  for (int ch = begin; ch < end; ++ch) {
    const int t0 = ch * C, rows = min(C, n - t0), t1 = t0 + C;
    const bool more = ch + 1 < end;
    const Gates& gates = s.s.gates[PASS == ALONE ? ch & 1 : 0];
    if (!AHEAD) {
      fk.load(k.at(t0), k.step, rows, tid);
      fq.load(q.at(t0), q.step, rows, tid);
      fv.load(v.at(t0), v.step, rows, tid, col);
    }
    __syncthreads();               // the chunk before is done with LDS
    fk.store(s.k, rows, tid);
    if (OUT) fq.store(s.q, rows, tid);
    if (!unit) fv.store(s.v, rows, tid);
    if constexpr (PASS != ALONE) fs.store(s.s, tid);
    if (more) {
      if (AHEAD) {
        fk.load(k.at(t1), k.step, n - t1, tid);
        if (OUT) fq.load(q.at(t1), q.step, n - t1, tid);
        if (!unit) fv.load(v.at(t1), v.step, n - t1, tid, col);
      }
      if (PASS != ALONE) fs.load(a.work, (int64_t)eh * chunks + ch + 1, tid);
      else if (w == 0) raw = load_gates(gate, t1, n - t1, lane);
    }
    __syncthreads();
    if constexpr (PASS == ALONE) solve_chunk<T, DK, NW, false>(s, gates, a.scale, lane, w);

    if (ks) {
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(ks + (int64_t)ch * DK * all + 256 * d) = S[d];
    }
    // K S and Q S
    f32x4 x[4], o[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] = o[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      WideOf<T, 3> sw;
      split(sw, join(S[2 * c], S[2 * c + 1]));
      Frag<T> kf[4], qf[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        kf[b] = load_tile(s.k + (16 * b + m) * LD, 32 * c, g);
        if (OUT) qf[b] = load_tile(s.q + (16 * b + m) * LD, 32 * c, g);
      }
      mma_all<T>(x, kf, sw);
      if (OUT) mma_all<T>(o, qf, front(sw));
    }
    f32x4 vs[4] = {};
    if (!unit) fv.get(vs, s.v, rows, w, lane);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 in = *reinterpret_cast<const f32x4*>(&gates.in[16 * b + 4 * g]);
      x[b] = vs[b] - in * x[b];
      o[b] *= in * a.scale;
    }
    if (PASS == ALONE) {
      if (w == 0 && more) make_gates(s.s.gates[(ch + 1) & 1], raw, gate.half, lane);
      __syncthreads();             // the inverses are there
    }
    f32x4 W[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
      for (int u = 0; u < b; ++u)
        mma16(x[b], *reinterpret_cast<const f32x4*>(&s.s.n[s.s.tile(b, u) + m * IP + 4 * g]), W[u]);
      W[b] = f32x4{0, 0, 0, 0};
      mma16(W[b], *reinterpret_cast<const f32x4*>(&s.s.inv[(16 * b + m) * IP + 4 * g]), x[b]);
    }
    if (kw) {
#pragma unroll
      for (int b = 0; b < 4; ++b) *reinterpret_cast<f32x4*>(kw + (int64_t)ch * C * all + 256 * b) = W[b];
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) W[b] *= *reinterpret_cast<const f32x4*>(&gates.beta[16 * b + 4 * g]);   // U
    if constexpr (OUT) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        WideOf<T, 2> uw;
        split(uw, join(W[2 * c], W[2 * c + 1]));
#pragma unroll
        for (int b = 2 * c; b < 4; ++b) mma<T>(o[b], s.s.p_row(16 * b + m, 32 * c, g), uw);
      }
    }
    if (OUT) fv.put(s.v, o, out.at(t0), out.step, rows, min(C, a.steps - t0), w, lane);
#pragma unroll
    for (int d = 0; d < DT; ++d) S[d] *= gates.across;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f32x4 u[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) u[i] = W[2 * c + i] * *reinterpret_cast<const f32x4*>(&gates.out[16 * (2 * c + i) + 4 * g]);
      WideOf<T, 3> uw;
      split(uw, join(u[0], u[1]));
      Frag<T> kf[DT];
#pragma unroll
      for (int d = 0; d < DT; ++d) kf[d] = load_col(s.k, LD, 32 * c, 16 * d, lane);
      mma_all<T>(S, kf, uw);
    }
    if (OUT) fv.write(s.v, out.at(t0), out.step, rows, min(C, a.steps - t0), w, lane);
  }
  if (!OUT) {
    put_carry<DT>(boundary(seg, eh, part, DK, all), S, unit, all, c0, w, lane);
    return;
  }
  const int to = PASS == ALONE || at + 1 == seg.count ? a.steps : (begin + seg.chunks) * C;
  for (int t = max(live, begin) * C + tid / DV; t < to; t += NT / DV) out.at(t)[tid % DV] = (T)0.0f;   // padding
  if (a.final_state && end == live && (begin < end || at == 0)) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.final_state[((int64_t)eh * DK + 16 * d + 4 * g + r) * all + c0 + col] = S[d][r];
  }
}

// ---- backward along the rollout ------------------------------------------------------------
// The gradient of the state, from the last chunk to the first, and with it M and v'.  Every
// product's columns are value columns, so a wave works on its 16 alone, as in the forward pass, and the
// same bounds it: 190 us at 512 x 300 bf16, 84 us at 512 x 50 fp32.
template <class T, int DK, int NW, Pass PASS>
__global__ __launch_bounds__(64 * NW, (PASS == ALONE ? waves_per_simd<T, DK, NW>() : PASS == CARRY && sizeof(T) == 2 ? 2 : 1)) void backward_state_kernel(bsg_delta a, Segments seg) {
  constexpr int LD = pitch<T>(DK), DT = DK / 16, DV = 16 * NW, NT = 64 * NW;
  // rows a chunk ahead; not for fp32 solved in place (600 envs x 50 steps, dims 32: 186 -> 198 us)
  constexpr bool AHEAD = PASS != ALONE || sizeof(T) == 2;
  constexpr bool OUT = PASS != CARRY, LDS = sizeof(T) == 2;
  __shared__ __align__(16) Chunk<T, DK, NW, PASS == ALONE, true, LDS> s;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, m = lane & 15, g = lane >> 4;
  // the workgroup's columns of all (CARRY: and of the unit matrix's, behind them) and its segment
  const int all = PASS == ALONE ? DV : a.dim_v, groups = all / DV + (OUT ? 0 : (DK + DV - 1) / DV);
  const int segments = PASS == ALONE ? 1 : OUT ? seg.count : seg.count - 1, id = blockIdx.x / groups, part = id % segments;
  const int eh = id / segments, h = eh % a.heads_v, e = eh / a.heads_v, hk = h / (a.heads_v / a.heads_k);
  const bool unit = !OUT && (int)(blockIdx.x % groups) >= all / DV;
  const int c0 = (int)(blockIdx.x % groups) * DV - (unit ? all : 0), col = 16 * w + m;
  const int n = steps_of(a, e), chunks = (a.steps + C - 1) / C, live = (n + C - 1) / C;
  const int at = OUT ? part : part + 1;              // the segment
  const int begin = PASS == ALONE ? 0 : at * seg.chunks, end = PASS == ALONE ? live : min(begin + seg.chunks, live);
  if (!OUT && (part + 1) * seg.chunks >= live) return;   // no boundary before the rollout's end

  constexpr int SIDE = PASS == JOINED ? DT : 2;          // tiles of D side by side: registers allow no more
  f32x4 D[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      D[d][r] = !OUT ? unit && 16 * d + 4 * g + r == c0 + col ? 1.0f : 0.0f
                     : a.dfinal ? a.dfinal[((int64_t)eh * DK + 16 * d + 4 * g + r) * all + c0 + col] : 0.0f;
  if (PASS == JOINED && end < live) {
    const float* p = tiles(boundary(seg, eh, at, DK, all), 0, 1, DT, c0 / 16 + w, lane);
#pragma unroll
    for (int d = 0; d < DT; ++d) D[d] = *reinterpret_cast<const f32x4*>(p + 256 * d);
  }

  Fetch<T, C, DK, NT> fk, fq;
  Columns<T, NW, LDS> fv;
  FetchSolved<T, NT, true> fs;
  RawGates raw = {0, 0, 0};
  const Steps<const T> k = steps_in<const T>(a.k, e, hk), q = steps_in<const T>(a.q, e, hk), dout = steps_in<const T>(a.dout, e, h, unit ? 0 : c0);
  const Steps<T> dv = steps_in<T>(a.dv, e, h, c0);
  const GateSteps gate(a, e, h);
  float *const ws = tiles(a.work_states, (int64_t)eh * chunks, all / 16, DT, c0 / 16 + w, lane), *const wm = tiles(a.work_w, (int64_t)eh * chunks, all / 16, 4, c0 / 16 + w, lane);
  if (begin < end) {
    const int t0 = (end - 1) * C;
    if (AHEAD) {
      fk.load(k.at(t0), k.step, n - t0, tid);
      if (!unit) {
        fq.load(q.at(t0), q.step, n - t0, tid);
        fv.load(dout.at(t0), dout.step, n - t0, tid, col);
      }
    }
    if constexpr (PASS != ALONE) {
      fs.load(a.work, (int64_t)eh * chunks + end - 1, tid);
    } else {
      if (w == 0) make_gates(s.s.gates[(end - 1) & 1], load_gates(gate, t0, n - t0, lane), gate.half, lane);
      clear_above(s.s, tid, NT);
    }
  }
  for (int ch = end - 1; ch >= begin; --ch) {
    const int t0 = ch * C, rows = min(C, n - t0), t1 = t0 - C;
    const bool more = ch > begin;
    const Gates& gates = s.s.gates[PASS == ALONE ? ch & 1 : 0];
    if (!AHEAD) {
      fk.load(k.at(t0), k.step, rows, tid);
      fq.load(q.at(t0), q.step, rows, tid);
      fv.load(dout.at(t0), dout.step, rows, tid, col);
    }
    __syncthreads();               // the chunk after is done with LDS
    fk.store(s.k, rows, tid);
    if (!unit) {
      fq.store(s.q, rows, tid);
      fv.store(s.v, rows, tid);
    }
    if constexpr (PASS != ALONE) fs.store(s.s, tid);
    if (more) {
      if (AHEAD) {
        fk.load(k.at(t1), k.step, C, tid);
        if (!unit) {
          fq.load(q.at(t1), q.step, C, tid);
          fv.load(dout.at(t1), dout.step, C, tid, col);
        }
      }
      if (PASS != ALONE) fs.load(a.work, (int64_t)eh * chunks + ch - 1, tid);
      else if (w == 0) raw = load_gates(gate, t1, C, lane);
    }
    __syncthreads();
    if constexpr (PASS == ALONE) solve_chunk<T, DK, NW, true>(s, gates, a.scale, lane, w);

    if (OUT)
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(ws + (int64_t)ch * DK * all + 256 * d) = D[d];

    f32x4 x[4], go[4] = {};
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] = f32x4{0, 0, 0, 0};
    if (!unit) fv.get(go, s.v, rows, w, lane);
#pragma unroll
    for (int c = 0; c < DK / 32; ++c) {
      WideOf<T, 3> dw;
      split(dw, join(D[2 * c], D[2 * c + 1]));
      Frag<T> kf[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) kf[b] = load_tile(s.k + (16 * b + m) * LD, 32 * c, g);
      mma_all<T>(x, kf, dw);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) x[b] *= *reinterpret_cast<const f32x4*>(&gates.out[16 * b + 4 * g]);
    if (!unit)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> gf = round_frag<T>(join(go[2 * c], go[2 * c + 1]));   // as it was read
#pragma unroll
        for (int b = 0; b < 2 * c + 2; ++b) mma<T>(x[b], s.s.p_col(16 * b, 32 * c, lane), gf);
      }
    if (PASS == ALONE) {
      if (w == 0 && more) make_gates(s.s.gates[(ch + 1) & 1], raw, gate.half, lane);
      __syncthreads();             // the inverses are there
    }
    f32x4 M[4];
#pragma unroll
    for (int b = 3; b >= 0; --b) {
#pragma unroll
      for (int u = b + 1; u < 4; ++u) {
        const float* p = &s.s.n[s.s.tile(u, b) + 4 * g * IP + m];
        mma16(x[b], f32x4{p[0], p[IP], p[2 * IP], p[3 * IP]}, M[u]);
      }
      const float* p = &s.s.inv[(16 * b + 4 * g) * IP + m];
      M[b] = f32x4{0, 0, 0, 0};
      mma16(M[b], f32x4{p[0], p[IP], p[2 * IP], p[3 * IP]}, x[b]);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (OUT) *reinterpret_cast<f32x4*>(wm + (int64_t)ch * C * all + 256 * b) = M[b];
      M[b] *= *reinterpret_cast<const f32x4*>(&gates.beta[16 * b + 4 * g]);
    }
    if (OUT) fv.put(s.v, M, dv.at(t0), dv.step, rows, min(C, a.steps - t0), w, lane);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 in = *reinterpret_cast<const f32x4*>(&gates.in[16 * b + 4 * g]);
      M[b] *= -in;
      go[b] *= in * a.scale;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) D[d] *= gates.across;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      WideOf<T, 3> lw, ow;
      split(lw, join(M[2 * c], M[2 * c + 1]));
      split(ow, join(go[2 * c], go[2 * c + 1]));
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += SIDE) {
        f32x4 x[SIDE];
        Frag<T> kf[SIDE], qf[SIDE];
#pragma unroll
        for (int d = 0; d < SIDE; ++d) {
          x[d] = D[d0 + d];
          kf[d] = load_col(s.k, LD, 32 * c, 16 * (d0 + d), lane);
          if (!unit) qf[d] = load_col(s.q, LD, 32 * c, 16 * (d0 + d), lane);
        }
        mma_all<T>(x, kf, lw);
        if (!unit) mma_all<T>(x, qf, ow);
#pragma unroll
        for (int d = 0; d < SIDE; ++d) D[d0 + d] = x[d];
      }
    }
    if (OUT) fv.write(s.v, dv.at(t0), dv.step, rows, min(C, a.steps - t0), w, lane);
  }
  if (!OUT) {
    put_carry<DT>(boundary(seg, eh, part, DK, all), D, unit, all, c0, w, lane);
    return;
  }
  const int to = PASS == ALONE || at + 1 == seg.count ? a.steps : (begin + seg.chunks) * C;
  for (int t = max(live, begin) * C + tid / DV; t < to; t += NT / DV) dv.at(t)[tid % DV] = (T)0.0f;   // padding
  if (a.dstate && at == 0) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.dstate[((int64_t)eh * DK + 16 * d + 4 * g + r) * all + c0 + col] = D[d][r];
  }
}

// ---- backward inside the chunks ------------------------------------------------------------
// q', k', beta', g' of one chunk, env and key head, all chunks side by side: a wave owns 16 steps.
// The matrices o'.w and m.w are needed by rows (for q', kr') and by columns (for kw'); both are
// computed, each in the layout in which it is the B operand of what follows, which costs less than
// a turn through LDS, by different waves.  Bound by memory: S, D, W, M and the rows of a chunk and head, 104 KB
// in dims 64, once (164 us a launch at 512 x 300, 3.3 TB/s).  The value dimension is walked in slices of 32.  Value heads
// that share a key head take a launch each: all but the last leave their sums of q' and k' in fp32 to
// the next (in one launch their sums cost the registers that let two workgroups share a CU: 420 us
// against 2 x 164 us, two heads to a key head, 512 envs x 300 steps).
constexpr int SL = 32;
template <class T, int R>
struct WideRows {                  // an R x SL tile of fp32 values as operand parts of type T
  static constexpr int n = Parts<T, 2>::n, LD = pitch<T>(SL);
  T p[n][R * LD];
  // lane l's part of D tile d (rows) of column block b
  __device__ __forceinline__ void put(int d, int b, int l, f32x4 x) {
    T* at = &p[0][(16 * d + 4 * (l >> 4)) * LD + 16 * b + (l & 15)];
#pragma unroll
    for (int i = 0; i < n; ++i, at += R * LD)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const T z = (T)x[r];
        at[r * LD] = z;
        x[r] -= (float)z;
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
  T k[C * pitch<T>(DK)], q[C * pitch<T>(DK)];
  union {
    struct {
      T go[C * pitch<T>(SL)];
      WideRows<T, C> w, mu;
      WideRows<T, DK> st, ds;
    };
    float kw[C * (DK + 4)];        // at the end: kw', on its way to the waves that hold kr'
  };
  Gates gates;
  float dc[2][C], part[8];
};

// Eight waves: 0..3 hold the 16 steps of tile w as they read the state (q', kr'), 4..7 those of tile
// w - 4 as they write it (kw').  The two run code of their own between the same barriers, so that
// neither pays for the other's registers: two workgroups to a CU where LDS holds two (four waves a
// SIMD cover each other's loads), else one, which loads a slice ahead.
template <class T, int DK> constexpr bool two_groups() { return 2 * sizeof(Inside<T, DK>) <= 160 * 1024; }

template <class T, int DK, bool READER>
__device__ __forceinline__ void chunk_gradient(Inside<T, DK>& s, float* sums, int head, int ch, int hk, int e) {
  constexpr int LD = pitch<T>(DK), DT = DK / 16, GL = pitch<T>(SL), NT = 512;
  constexpr int NS = DK * SL / 4 / NT > 0 ? DK * SL / 4 / NT : 1;   // f32x4 of a state's slice to a thread
  constexpr bool AHEAD = !two_groups<T, DK>();
  static_assert(C * SL / 4 == NT, "one f32x4 of W and of M to a thread");
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), own = 16 * (w & 3) + m, tile = w & 3;
  const bsg_delta& a = arguments();
  const int chunks = (a.steps + C - 1) / C, group = a.heads_v / a.heads_k, DV = a.dim_v, h = hk * group + head;
  const int t0 = ch * C, rows = min(C, steps_of(a, e) - t0);
  const float scale = a.scale;
  const bool half = a.gate_dtype == BSG_BF16;

  // one slice on its way from memory to LDS
  constexpr int GV = Vec<T>::n, GROW = SL / GV;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 fgo = {0, 0, 0, 0};
  f32x4 fw, fm, fs[NS], fd[NS];
  const auto fetch = [&](int v0) {
    const bsg_delta& a = arguments();
    const int64_t ehc = ((int64_t)e * a.heads_v + h) * chunks + ch;
    const int64_t at = ehc * C * DV + v0 * C + tid * 4, as = ehc * DK * DV + v0 * DK + tid * 4;
    if (tid < C * GROW)
      fgo = *reinterpret_cast<const u32x4*>(row<T>(a.dout, e, t0 + min(tid / GROW, rows - 1), h) + v0 + tid % GROW * GV);
    fw = *reinterpret_cast<const f32x4*>(a.kept_w + at);
    fm = *reinterpret_cast<const f32x4*>(a.work_w + at);
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (DK * SL / 4 >= NT || tid < DK * SL / 4) {
        fs[i] = *reinterpret_cast<const f32x4*>(a.kept_states + as + i * 4 * NT);
        fd[i] = *reinterpret_cast<const f32x4*>(a.work_states + as + i * 4 * NT);
      }
  };
  if (AHEAD) fetch(0);

  // readers: o'.w and m.w by rows j, q' and kr'; writers: by rows i, kw'
  f32x4 ow[4], mw[4], X1[DT], X2[DT];
#pragma unroll
  for (int b = 0; b < 4; ++b) ow[b] = mw[b] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < DT; ++d) X1[d] = X2[d] = f32x4{0, 0, 0, 0};
  float dbeta = 0.0f, sd = 0.0f;
  RawGates raw = {0, 0, 0};
  if (READER && w == 0) raw = load_gates(GateSteps(arguments(), e, h), t0, rows, lane);
  for (int v0 = 0; v0 < DV; v0 += SL) {
    if (!AHEAD) fetch(v0);
    __syncthreads();             // the slice before is done with
    if (READER && v0 == 0 && w == 0) make_gates(s.gates, raw, half, lane);
    if (tid < C * GROW)
      *reinterpret_cast<u32x4*>(&s.go[tid / GROW * GL + tid % GROW * GV]) = tid / GROW < rows ? fgo : u32x4{0, 0, 0, 0};
    s.w.put(tid / 64 % 4, tid / 256, lane, fw);
    s.mu.put(tid / 64 % 4, tid / 256, lane, fm);
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (DK * SL / 4 >= NT || tid < DK * SL / 4) {
        const int at = (tid + i * NT) / 64;
        s.st.put(at % DT, at / DT, lane, fs[i]);
        s.ds.put(at % DT, at / DT, lane, fd[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) sd = fmaf(fs[i][j], fd[i][j], sd);
      }
    if (AHEAD) {
      if (v0 + SL < DV) fetch(v0 + SL);
    }
    __syncthreads();
    const WideOf<T, 2> wf = s.w.get(own, g);
    if (READER) {
      const Frag<T> go = load_run(s.go + own * GL, 0, g);
      const WideOf<T, 2> mf = s.mu.get(own, g);
      const f32x8 wx = whole(wf), mx = whole(mf);
#pragma unroll
      for (int j = 0; j < 8; ++j) dbeta = fmaf(wx[j], mx[j], dbeta);
      // (bf16: tiles behind the own one too: cheaper than a branch, and masked below)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (sizeof(T) == 4 && b > tile) continue;
        const WideOf<T, 2> x = s.w.get(16 * b + m, g);
        mma<T>(ow[b], x, go);
        mma<T>(mw[b], x, mf);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const WideOf<T, 2> x = s.st.get(16 * d + m, g);
        mma<T>(X1[d], x, go);
        mma<T>(X2[d], x, mf);
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (sizeof(T) == 4 && b < tile) continue;
        mma<T>(ow[b], load_run(s.go + (16 * b + m) * GL, 0, g), wf);
        mma<T>(mw[b], s.mu.get(16 * b + m, g), wf);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) mma<T>(X1[d], s.ds.get(16 * d + m, g), wf);
    }
  }
  // scale by the gates of the wave's own step (its lane) and add the chunk's own terms
  const Gates& G = s.gates;
  const Step me = step_of(G, own);
  const float bi = G.beta[own], in = G.in[own], out = G.out[own], across = G.across;
  float y = 0.0f, dc = 0.0f;
  if (READER) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      X1[d] *= in;
      X2[d] *= in;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (2 * c <= tile) {       // rows j of tiles 2c, 2c + 1 against the own step i
        f32x4 f1[2], f2[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 16 * (2 * c + u) + 4 * g;
          const f32x4 f = decays<true>(G, row, me) * *reinterpret_cast<const f32x4*>(&G.beta[row]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f1[u][r] = row + r <= own ? f[r] * ow[2 * c + u][r] : 0.0f;
            f2[u][r] = row + r < own ? f[r] * mw[2 * c + u][r] : 0.0f;
          }
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
  } else {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 k = widen(*reinterpret_cast<const Half<T>*>(&s.k[own * LD + 16 * d + 4 * g]));
      X1[d] *= out;
#pragma unroll
      for (int r = 0; r < 4; ++r) y = fmaf(k[r], X1[d][r], y);
    }
    y *= bi;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (2 * c + 1 >= tile) {   // rows i of tiles 2c, 2c + 1 against the own step j
        f32x4 f1[2], f2[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int row = 16 * (2 * c + u) + 4 * g;
          const f32x4 f = decays<false>(G, row, me), bm = f * *reinterpret_cast<const f32x4*>(&G.beta[row]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f1[u][r] = row + r >= own ? scale * f[r] * ow[2 * c + u][r] : 0.0f;
            f2[u][r] = row + r > own ? -bm[r] * mw[2 * c + u][r] : 0.0f;
          }
        }
        WideOf<T, 2> w1, w2;
        split(w1, join(f1[0], f1[1]));
        split(w2, join(f2[0], f2[1]));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          mma<T>(X1[d], load_col(s.q, LD, 32 * c, 16 * d, lane), w1);
          mma<T>(X1[d], load_col(s.k, LD, 32 * c, 16 * d, lane), w2);
        }
      }
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const f32x4 k = widen(*reinterpret_cast<const Half<T>*>(&s.k[own * LD + 16 * d + 4 * g]));
    X1[d] *= READER ? scale : bi;
    if (READER) {
      const f32x4 q = widen(*reinterpret_cast<const Half<T>*>(&s.q[own * LD + 16 * d + 4 * g]));
      X2[d] *= -bi;
#pragma unroll
      for (int r = 0; r < 4; ++r) dc = fmaf(q[r], X1[d][r], fmaf(k[r], X2[d][r], dc));
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) dc = fmaf(-k[r], X1[d][r], dc);
    }
  }
  dc = sum_groups(dc);
  // the chunk's last step: across <S, D> + sum_j k_j.(out_j D u_j)
  y += across * sd;
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) y += __shfl_xor(y, d);
  if (g == 0) s.dc[READER ? 0 : 1][own] = dc;
  if (lane == 0) s.part[w] = y;
  const bsg_delta& z = arguments();
  if (READER) {
    dbeta = sum_groups(dbeta);
    if (g == 0 && t0 + own < z.steps) gate_out(z.dbeta, z.gate_dtype, e, t0 + own, h, own < rows ? dbeta : 0.0f);
  }
  __syncthreads();
  if (READER && w == 0) {
    float x = s.dc[0][lane] + s.dc[1][lane];
    if (lane == 63)
#pragma unroll
      for (int i = 0; i < 8; ++i) x += s.part[i];
    const int ep = G.episode[lane], before = lane ? G.episode[lane - 1] : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const float o = __shfl_down(x, d);
      const int oe = __shfl_down(ep, d);
      if (lane + d < 64 && oe == ep) x += o;
    }
    // a first step's decay meets no state
    if (t0 + lane < z.steps)
      gate_out(z.dg, z.gate_dtype, e, t0 + lane, h, lane < rows && ep == before ? x : 0.0f);
  }
  if (!READER) {                   // the last slice is done with: every wave has passed the barrier above
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&s.kw[own * (DK + 4) + 16 * d + 4 * g]) = X1[d];
  }
  __syncthreads();
  if (!READER) return;
  // 16 bytes a lane of the sums over the heads before, as the D tiles lie
  float* sum = sums ? sums + ((((int64_t)e * z.heads_k + hk) * chunks + ch) * 4 + tile) * 2 * DT * 256 + lane * 4 : nullptr;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    X2[d] += *reinterpret_cast<const f32x4*>(&s.kw[own * (DK + 4) + 16 * d + 4 * g]);
    if (sum && head > 0) {
      X1[d] += *reinterpret_cast<const f32x4*>(sum + 512 * d);
      X2[d] += *reinterpret_cast<const f32x4*>(sum + 512 * d + 256);
    }
  }
  if (head + 1 < group) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      *reinterpret_cast<f32x4*>(sum + 512 * d) = X1[d];
      *reinterpret_cast<f32x4*>(sum + 512 * d + 256) = X2[d];
    }
    return;
  }
  if (t0 + own >= z.steps) return;
  T *oq = row_out<T>(z.dq, e, t0 + own, hk), *ok = row_out<T>(z.dk, e, t0 + own, hk);
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    store4(oq + 16 * d + 4 * g, own < rows ? X1[d] : f32x4{0, 0, 0, 0});
    store4(ok + 16 * d + 4 * g, own < rows ? X2[d] : f32x4{0, 0, 0, 0});
  }
}

template <class T, int DK>
__global__ __launch_bounds__(512, (two_groups<T, DK>() ? 4 : 2)) void backward_chunk_kernel(bsg_delta, float* sums, int head) {
  constexpr int NT = 512;
  __shared__ __align__(16) Inside<T, DK> s;
  const bsg_delta& a = arguments();
  const int tid = threadIdx.x, chunks = (a.steps + C - 1) / C, group = a.heads_v / a.heads_k;
  const int ch = blockIdx.x % chunks, ehk = blockIdx.x / chunks, hk = ehk % a.heads_k, e = ehk / a.heads_k;
  const int t0 = ch * C, rows = min(C, steps_of(a, e) - t0), all = min(C, a.steps - t0);
  if (rows <= 0) {                 // padding
    if (head > 0) return;
    const Steps<T> dqs = steps_in<T>(a.dq, e, hk), dks = steps_in<T>(a.dk, e, hk);
    for (int i = tid; i < all * DK; i += NT) dqs.at(t0 + i / DK)[i % DK] = dks.at(t0 + i / DK)[i % DK] = (T)0.0f;
    for (int i = tid; i < all * group; i += NT) {
      gate_out(a.dg, a.gate_dtype, e, t0 + i / group, hk * group + i % group, 0.0f);
      gate_out(a.dbeta, a.gate_dtype, e, t0 + i / group, hk * group + i % group, 0.0f);
    }
    return;
  }
  {
    Fetch<T, C, DK, NT> fk, fq;
    fk.load(row<T>(a.k, e, t0, hk), a.k.step, rows, tid);
    fq.load(row<T>(a.q, e, t0, hk), a.q.step, rows, tid);
    fk.store(s.k, rows, tid);
    fq.store(s.q, rows, tid);
  }
  if (__builtin_amdgcn_readfirstlane(tid >> 6) < 4) chunk_gradient<T, DK, true>(s, sums, head, ch, hk, e);
  else chunk_gradient<T, DK, false>(s, sums, head, ch, hk, e);
}

// ---- acting --------------------------------------------------------------------------------
// One wave per env, value head and slice of value columns: the slice of the state in registers,
// both sums over it (S^T k and S^T q) in one pass, then the update.  Lanes hold four columns;
// S'^T q = (S + k u^T)^T q = S^T q + (k.q) u.  The state is read and written once, at the rate of a large
// copy: 4096 envs, 4 heads, 64 x 64 in 105-109 us a call for 537 MB.
template <class T, int DK, int DV>
__global__ __launch_bounds__(256) void step_kernel(bsg_delta_act a, int64_t waves) {
  constexpr int COLS = DV == 32 || DK == 128 ? 32 : 64, L = COLS / 4, RG = 64 / L, N = DK / RG, SLICES = DV / COLS;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= waves) return;
  const int lane = threadIdx.x & 63, rg = lane / L;
  const int64_t eh = id / SLICES;
  const int c0 = (int)(id % SLICES) * COLS + lane % L * 4;
  const int h = (int)(eh % a.heads_v), e = (int)(eh / a.heads_v), hk = h / (a.heads_v / a.heads_k);
  const bool first = a.first && a.first[e * a.first_env] != 0;
  float* st = a.state + eh * DK * DV + c0;
  f32x4 S[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    S[i] = first ? f32x4{0, 0, 0, 0} : *reinterpret_cast<const f32x4*>(st + (i * RG + rg) * DV);
  const T *kr = row<T>(a.k, e, 0, hk), *qr = row<T>(a.q, e, 0, hk);
  const f32x4 v = widen(*reinterpret_cast<const Half<T>*>(row<T>(a.v, e, 0, h) + c0));
  const float alpha = expf(at_least_lowest(gate(a.g, a.gate_dtype, e, 0, h))), beta = gate(a.beta, a.gate_dtype, e, 0, h);
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


template <class T, int DK, int NW>
hipError_t run(const bsg_delta_act& a, bool, hipStream_t st) {
  constexpr int DV = 16 * NW, slices = DV / (DV == 32 || DK == 128 ? 32 : 64);
  const int64_t waves = (int64_t)a.num_envs * a.heads_v * slices;
  step_kernel<T, DK, DV><<<dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st>>>(a, waves);
  return hipGetLastError();
}
// Where the rows (envs x value heads) leave CUs idle, the pass along a rollout is bound by the time
// of one chunk, and the chunks are solved beforehand, side by side; where they do not, solving
// in place saves the way of the matrices through memory.
bool solved_first(const bsg_delta& a) {
  return a.dim_v > 32 && a.steps > C && (int64_t)a.num_envs * a.heads_v < 256;
}
int64_t solved_work(const bsg_delta& a) {
  if (!solved_first(a)) return 0;
  const int64_t chunks = (int64_t)a.num_envs * a.heads_v * ((a.steps + C - 1) / C);
  return chunks * (a.dtype == BSG_BF16 ? solved_bytes<bf16>() : solved_bytes<float>());
}
// ... and the rollout is cut into as many segments as give each CU a workgroup of the last pass, of three
// chunks at least (a boundary costs its transition and its turn of the join).  Learning call, 4 heads, dim
// 128: 4 envs x 4095 steps 854 -> 422 us, 1 x 4095 743 -> 232, 8 x 4095 1001 -> 740, 4 x 1000 238 -> 178,
// 2 x 700 180 -> 161; at 500 steps the host's time for the launches takes what it saves (183 -> 198).
// Two workgroups a CU: 4 x 4095 462 us; two segments: 16 x 4095 1327 -> 1288 us, hence three at least.
Segments segments(const bsg_delta& a) {
  const int chunks = (a.steps + C - 1) / C, rows = a.num_envs * a.heads_v;
  Segments seg = {nullptr, 1, chunks};
  if (!solved_first(a)) return seg;
  const int most = min(256 / (rows * (a.dim_v / 64)), chunks / 3);
  if (most < 3) return seg;
  seg.chunks = (chunks + most - 1) / most;
  seg.count = (chunks + seg.chunks - 1) / seg.chunks;
  seg.carry = reinterpret_cast<float*>(static_cast<char*>(a.work) + solved_work(a));
  return seg;
}
int64_t carry_work(const bsg_delta& a) {
  return (int64_t)a.num_envs * a.heads_v * (segments(a).count - 1) * a.dim_k * (a.dim_k + a.dim_v) * 4;
}
template <class T, int DK, int NW>
hipError_t run(const bsg_delta& a, bool back, hipStream_t st) {
  const dim3 rows((unsigned)(a.num_envs * a.heads_v));
  const Segments seg = segments(a);
  if (solved_first(a)) {
    if constexpr (NW > 2) {
      const dim3 all((unsigned)(rows.x * ((a.steps + C - 1) / C))), groups(rows.x * (NW / 4) * seg.count);
      const dim3 carries(rows.x * (NW / 4 + (DK + 63) / 64) * (seg.count - 1)), joins(rows.x * NW);
      if (back) {
        solve_kernel<T, DK, true><<<all, dim3(256), 0, st>>>(a);
        if (seg.count > 1) {
          backward_state_kernel<T, DK, 4, CARRY><<<carries, dim3(256), 0, st>>>(a, seg);
          join_kernel<DK, true><<<joins, dim3(4 * DK), 0, st>>>(a, seg);
        }
        backward_state_kernel<T, DK, 4, JOINED><<<groups, dim3(256), 0, st>>>(a, seg);
      } else {
        solve_kernel<T, DK, false><<<all, dim3(256), 0, st>>>(a);
        if (seg.count > 1) {
          forward_kernel<T, DK, 4, CARRY><<<carries, dim3(256), 0, st>>>(a, seg);
          join_kernel<DK, false><<<joins, dim3(4 * DK), 0, st>>>(a, seg);
        }
        forward_kernel<T, DK, 4, JOINED><<<groups, dim3(256), 0, st>>>(a, seg);
      }
    }
  } else if (back) {
    backward_state_kernel<T, DK, NW, ALONE><<<rows, dim3(64 * NW), 0, st>>>(a, seg);
  } else {
    forward_kernel<T, DK, NW, ALONE><<<rows, dim3(64 * NW), 0, st>>>(a, seg);
  }
  if (back) {
    const dim3 chunks((unsigned)(a.num_envs * a.heads_k * ((a.steps + C - 1) / C)));
    const int group = a.heads_v / a.heads_k;
    float* sums = group > 1 ? reinterpret_cast<float*>(static_cast<char*>(a.work) + solved_work(a) + carry_work(a)) : nullptr;
    for (int head = 0; head < group; ++head) backward_chunk_kernel<T, DK><<<chunks, dim3(512), 0, st>>>(a, sums, head);
  }
  return hipGetLastError();
}
template <class T, int DK, class A>
hipError_t run(const A& a, bool back, hipStream_t st) {
  return a.dim_v == 32 ? run<T, DK, 2>(a, back, st) : a.dim_v == 64 ? run<T, DK, 4>(a, back, st) : run<T, DK, 8>(a, back, st);
}
template <class T, class A>
hipError_t run(const A& a, bool back, hipStream_t st) {
  return a.dim_k == 32 ? run<T, 32>(a, back, st) : a.dim_k == 64 ? run<T, 64>(a, back, st) : run<T, 128>(a, back, st);
}
template <class A> hipError_t run(const A& a, bool back, hipStream_t st) {
  return a.dtype == BSG_BF16 ? run<bf16>(a, back, st) : run<float>(a, back, st);
}

}  // namespace

namespace bsg {

// Shapes, strides and pointers are validated by the bsg_delta_* entry points (bsg_abi.cpp).
hipError_t launch_delta_forward(const bsg_delta& a, hipStream_t st) { return run(a, false, st); }
hipError_t launch_delta_backward(const bsg_delta& a, hipStream_t st) { return run(a, true, st); }
int64_t delta_work_bytes(const bsg_delta& a, bool back) {
  const int64_t chunks = (int64_t)a.num_envs * a.heads_k * ((a.steps + C - 1) / C);
  return solved_work(a) + carry_work(a) + (back && a.heads_v > a.heads_k ? chunks * C * a.dim_k * 2 * 4 : 0);
}
hipError_t launch_delta_step(const bsg_delta_act& a, hipStream_t st) { return run(a, false, st); }

}  // namespace bsg
