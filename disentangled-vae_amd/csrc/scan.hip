// The selective state-space scan, channels-last.  Per channel d with N states, token by token within a sequence:
//   dt    = softplus(delta + bias)                       (softplus optional)
//   h[n]  = exp(dt A[d,n]) h[n] + dt u B[n]              B, C shared by the channels of a group
//   out   = (sum_n C[n] h[n] + D u) * silu(z)            D and z optional
// States, step sizes and sums are fp32 whatever the activations' type; the output is rounded once.
//
// A lane owns one channel and keeps its N states in registers, so the sum over n is a chain of fused multiply-adds and
// neighbouring lanes read neighbouring channels.  B and C of a token are the same for all lanes: they come through the
// scalar unit and enter the vector instructions as scalar operands.
#include "seq_common.h"

#define SCAN_Q 8       // tokens per block: what is loaded ahead, and how far apart training keeps states
#define SCAN_MAX_N 16

struct ScanArgs {
  const void *u, *delta, *z, *B, *C, *dout;
  int64_t u_sb, u_st, delta_sb, delta_st, z_sb, z_st, B_sb, B_st, B_sg, C_sb, C_st, C_sg, dout_sb, dout_st;
  const float *A, *Dp, *bias, *state0;
  const float* dstate1;
  float *state1, *dstate0;
  void *out, *du, *ddelta, *dz;
  float *ckpt;                 // [row][block of SCAN_Q tokens][n][D]: the state that enters the block
  float *part_bc, *part_a;     // partial sums of the gradients of B and C, and of A, D and bias
  const int32_t* offsets;
  int rows, L, D, G, N, S, Dg, tpg, ntiles, softplus, blocks;
};

// what happens inside a block of n tokens from t0 on: bit j of `start` / `end` / `valid`: token t0 + j is its
// sequence's first / its sequence's last / in a sequence at all
struct Marks { uint32_t start, end, valid; };

template <bool PACKED>
__device__ __forceinline__ Marks block_marks(SeqWalk w, int t0, int n, int L) {
  Marks m = {0u, 0u, 0u};
  const uint32_t all = (1u << n) - 1u;
  if (!PACKED) {
    m.start = t0 == 0 ? 1u : 0u;
    m.end = t0 + n == L ? 1u << (n - 1) : 0u;
    m.valid = all;
    return m;
  }
  while (w.s < w.S && w.b < t0 + n) {
    if (w.b >= t0) m.start |= 1u << (w.b - t0);
    if (w.e <= t0 + n) m.end |= 1u << (w.e - 1 - t0);
    const uint32_t from = w.b > t0 ? ~0u << (w.b - t0) : ~0u;
    const uint32_t upto = w.e < t0 + n ? (1u << (w.e - t0)) - 1u : all;
    m.valid |= from & upto;
    if (w.e >= t0 + n) break;
    w.next(w.e);
  }
  return m;
}

// the N values of B or C at one token.  FAST: N == NP and 4-byte aligned, read as whole words
template <typename T, int NP, bool FAST> struct BCLoad;
template <int NP> struct BCLoad<float, NP, true> {
  static __device__ __forceinline__ void get(const float* p, int64_t off, int, float (&v)[NP]) {
#pragma unroll
    for (int n = 0; n < NP; ++n) v[n] = uniform_load(p + off, n);
  }
};
template <int NP> struct BCLoad<bf16_t, NP, true> {
  static __device__ __forceinline__ void get(const bf16_t* p, int64_t off, int, float (&v)[NP]) {
    const uint32_t* q = (const uint32_t*)(p + off);
#pragma unroll
    for (int n = 0; n < NP / 2; ++n) {
      const uint32_t w = uniform_load(q, n);
      v[2 * n] = __uint_as_float(w << 16);
      v[2 * n + 1] = __uint_as_float(w & 0xffff0000u);
    }
  }
};
template <typename T, int NP> struct BCLoad<T, NP, false> {
  static __device__ __forceinline__ void get(const T* p, int64_t off, int N, float (&v)[NP]) {
#pragma unroll
    for (int n = 0; n < NP; ++n) v[n] = n < N ? to_f32(p[off + n]) : 0.f;
  }
};

// One wave: 64 channels of one group of one row.
struct Tile {
  int g, d, lane, dl;
  bool on;
  __device__ __forceinline__ Tile(const ScanArgs& p, int tile) {
    lane = threadIdx.x & 63;
    g = tile / p.tpg;
    const int c = (tile % p.tpg) * 64 + lane;
    on = c < p.Dg;
    d = g * p.Dg + (on ? c : p.Dg - 1);          // lanes past the group's last channel read it too, and write nothing
  }
};

template <int NP>
__device__ __forceinline__ void load_state(const float* s, int64_t seq, const ScanArgs& p, int d, float (&h)[NP]) {
  const float* q = s + (seq * p.D + d) * p.N;
#pragma unroll
  for (int n = 0; n < NP; ++n) h[n] = n < p.N ? q[n] : 0.f;
}
template <int NP>
__device__ __forceinline__ void store_state(float* s, int64_t seq, const ScanArgs& p, int d, const float (&h)[NP]) {
  float* q = s + (seq * p.D + d) * p.N;
#pragma unroll
  for (int n = 0; n < NP; ++n)
    if (n < p.N) q[n] = h[n];
}
// the state that a sequence starts with
template <int NP>
__device__ __forceinline__ void entering_state(const ScanArgs& p, int64_t seq, int d, float (&h)[NP]) {
  if (p.state0) load_state<NP>(p.state0, seq, p, d, h);
  else {
#pragma unroll
    for (int n = 0; n < NP; ++n) h[n] = 0.f;
  }
}

template <typename T, int NP, bool PACKED, bool FAST>
__global__ void __launch_bounds__(256) scan_fwd_kernel(ScanArgs p) {
  const int wave = uniform(threadIdx.x >> 6);
  const int tgroups = (p.ntiles + 3) / 4;
  const int tile = (int)(blockIdx.x % tgroups) * 4 + wave;
  const int row = blockIdx.x / tgroups;
  if (tile >= p.ntiles) return;
  const Tile w(p, tile);
  float A2[NP], h[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] = n < p.N ? p.A[(int64_t)w.d * p.N + n] * LOG2E_F : 0.f;
    h[n] = 0.f;
  }
  const float Dp = p.Dp ? p.Dp[w.d] : 0.f, bias = p.bias ? p.bias[w.d] : 0.f;
  const T* u = (const T*)p.u + row * p.u_sb;
  const T* dl = (const T*)p.delta + row * p.delta_sb;
  const T* z = p.z ? (const T*)p.z + row * p.z_sb : nullptr;
  const T* B = (const T*)p.B + row * p.B_sb + w.g * p.B_sg;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  T* out = (T*)p.out + (int64_t)row * p.L * p.D;
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};
  if (PACKED) q.seek(0);

  for (int t0 = 0; t0 < p.L; t0 += SCAN_Q) {
    const int n = min(SCAN_Q, p.L - t0);
    const Marks m = block_marks<PACKED>(q, t0, n, p.L);
    if (p.ckpt && w.on) {
      float* ck = p.ckpt + ((int64_t)row * p.blocks + t0 / SCAN_Q) * p.N * p.D + w.d;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if (i < p.N) ck[(int64_t)i * p.D] = h[i];
    }
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int64_t t = t0 + j;
      if (!(m.valid >> j & 1)) {
        if (w.on) out[t * p.D + w.d] = from_f32<T>(0.f);
        continue;
      }
      if (m.start >> j & 1) entering_state<NP>(p, q.seq(), w.d, h);
      const float uu = to_f32(u[t * p.u_st + w.d]);
      const float pre = to_f32(dl[t * p.delta_st + w.d]) + bias;
      const float dt = p.softplus ? softplus_hw(pre) : pre;
      float Bv[NP], Cv[NP];
      BCLoad<T, NP, FAST>::get(B, t * p.B_st, p.N, Bv);
      BCLoad<T, NP, FAST>::get(C, t * p.C_st, p.N, Cv);
      const float x = dt * uu;
      float y = Dp * uu;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        h[i] = fmaf(exp2_hw(dt * A2[i]), h[i], x * Bv[i]);
        y = fmaf(Cv[i], h[i], y);
      }
      if (z) {
        const float zz = to_f32(z[t * p.z_st + w.d]);
        y *= zz * sigmoid_hw(zz);
      }
      if (w.on) out[t * p.D + w.d] = from_f32<T>(y);
      if (m.end >> j & 1) {
        if (p.state1 && w.on) store_state<NP>(p.state1, q.seq(), p, w.d, h);
        if (PACKED) q.next((int)t + 1);
      }
    }
  }
}

// The way back.  With g = dout silu(z), for a sequence's tokens from the last to the first:
//   dh[n]  = C[n] g + (a[n] dh[n] of the token behind)
//   dC[n] += g h[n]        dB[n] += dh[n] dt u          (sums over the group's channels)
//   w      = a[n] dh[n] (what goes on to the token before);  k = w h_before[n]
//   dA[n] += k dt          ddt += k A[n] + dh[n] B[n] u  du += dh[n] B[n] dt
// The states are computed again, SCAN_Q tokens at a time, from those that the forward pass kept.
template <typename T, int NP, bool PACKED, bool FAST>
__global__ void __launch_bounds__(256) scan_bwd_kernel(ScanArgs p) {
  const int wave = uniform(threadIdx.x >> 6);
  const int tgroups = (p.ntiles + 3) / 4;
  const int tile = (int)(blockIdx.x % tgroups) * 4 + wave;
  const int row = blockIdx.x / tgroups;
  if (tile >= p.ntiles) return;
  const Tile w(p, tile);
  const int tig = tile % p.tpg;
  float A2[NP], dh[NP], dA[NP], hs[SCAN_Q + 1][NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] = n < p.N ? p.A[(int64_t)w.d * p.N + n] * LOG2E_F : 0.f;
    dh[n] = dA[n] = 0.f;
  }
  float dD = 0.f, dbias = 0.f;
  const float Dp = p.Dp ? p.Dp[w.d] : 0.f, bias = p.bias ? p.bias[w.d] : 0.f;
  const T* u = (const T*)p.u + row * p.u_sb;
  const T* dl = (const T*)p.delta + row * p.delta_sb;
  const T* z = p.z ? (const T*)p.z + row * p.z_sb : nullptr;
  const T* go = (const T*)p.dout + row * p.dout_sb;
  const T* B = (const T*)p.B + row * p.B_sb + w.g * p.B_sg;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  const int64_t flat = (int64_t)row * p.L;
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};      // the sequence that the way back is in
  if (PACKED) { q.s = p.S; q.prev(p.L - 1); }

  for (int t0 = (p.L - 1) / SCAN_Q * SCAN_Q; t0 >= 0; t0 -= SCAN_Q) {
    const int n = min(SCAN_Q, p.L - t0);
    SeqWalk f = q;                                     // and the one that the states' second computation is in
    if (PACKED) f.seek(t0);
    const Marks m = block_marks<PACKED>(f, t0, n, p.L);
    const float* ck = p.ckpt + ((int64_t)row * p.blocks + t0 / SCAN_Q) * p.N * p.D + w.d;
#pragma unroll
    for (int i = 0; i < NP; ++i) hs[0][i] = i < p.N ? ck[(int64_t)i * p.D] : 0.f;
    float ub[SCAN_Q], pb[SCAN_Q], db[SCAN_Q];
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) {
#pragma unroll
      for (int i = 0; i < NP; ++i) hs[j + 1][i] = hs[j][i];
      if (!(m.valid >> j & 1)) continue;
      const int64_t t = t0 + j;
      ub[j] = to_f32(u[t * p.u_st + w.d]);
      pb[j] = to_f32(dl[t * p.delta_st + w.d]) + bias;
      db[j] = p.softplus ? softplus_hw(pb[j]) : pb[j];
      if (m.start >> j & 1) entering_state<NP>(p, f.seq(), w.d, hs[j + 1]);
      float Bv[NP];
      BCLoad<T, NP, FAST>::get(B, t * p.B_st, p.N, Bv);
      const float x = db[j] * ub[j];
#pragma unroll
      for (int i = 0; i < NP; ++i) hs[j + 1][i] = fmaf(exp2_hw(db[j] * A2[i]), hs[j + 1][i], x * Bv[i]);
      if (PACKED && (m.end >> j & 1)) f.next((int)t + 1);
    }
#pragma unroll
    for (int j = SCAN_Q - 1; j >= 0; --j) {
      if (j >= n) continue;
      const int64_t t = t0 + j, o = (flat + t) * p.D + w.d;
      if (!(m.valid >> j & 1)) {
        if (w.on) {
          ((T*)p.du)[o] = from_f32<T>(0.f);
          ((T*)p.ddelta)[o] = from_f32<T>(0.f);
          if (z) ((T*)p.dz)[o] = from_f32<T>(0.f);
        }
        for (int i = w.lane; i < 2 * p.N; i += 64)
          p.part_bc[(((int64_t)tig * p.rows * p.L + flat + t) * p.G + w.g) * 2 * p.N + i] = 0.f;
        continue;
      }
      if (m.end >> j & 1) {
        if (p.dstate1) load_state<NP>(p.dstate1, q.seq(), p, w.d, dh);
        else {
#pragma unroll
          for (int i = 0; i < NP; ++i) dh[i] = 0.f;
        }
      }
      float Bv[NP], Cv[NP];
      BCLoad<T, NP, FAST>::get(B, t * p.B_st, p.N, Bv);
      BCLoad<T, NP, FAST>::get(C, t * p.C_st, p.N, Cv);
      float g = w.on ? to_f32(go[t * p.dout_st + w.d]) : 0.f;
      if (z) {
        const float zz = to_f32(z[t * p.z_st + w.d]);
        const float sg = sigmoid_hw(zz);
        float y = Dp * ub[j];
#pragma unroll
        for (int i = 0; i < NP; ++i) y = fmaf(Cv[i], hs[j + 1][i], y);
        if (w.on) ((T*)p.dz)[o] = from_f32<T>(g * y * sg * fmaf(zz, 1.f - sg, 1.f));
        g *= zz * sg;
      }
      const float x = w.on ? db[j] * ub[j] : 0.f;
      float through = 0.f, ka = 0.f, pc[NP], pd[NP], hb[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) hb[i] = hs[j][i];
      if (m.start >> j & 1) entering_state<NP>(p, q.seq(), w.d, hb);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float a = exp2_hw(db[j] * A2[i]);
        const float d = fmaf(Cv[i], g, dh[i]);
        pc[i] = g * hs[j + 1][i];
        pd[i] = d * x;
        through = fmaf(d, Bv[i], through);
        dh[i] = d * a;
        const float k = dh[i] * hb[i];
        dA[i] = fmaf(k, db[j], dA[i]);
        ka = fmaf(k, A2[i], ka);
      }
      float* pb_ = p.part_bc + (((int64_t)tig * p.rows * p.L + flat + t) * p.G + w.g) * 2 * p.N;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float sb = wave_sum(pd[i]), sc = wave_sum(pc[i]);
        if (w.lane == 0 && i < p.N) { pb_[i] = sb; pb_[p.N + i] = sc; }
      }
      dD = fmaf(g, ub[j], dD);
      float dd = fmaf(ka, LN2_F, through * ub[j]);
      if (p.softplus) dd *= sigmoid_hw(pb[j]);
      dbias += dd;
      if (w.on) {
        ((T*)p.du)[o] = from_f32<T>(fmaf(through, db[j], Dp * g));
        ((T*)p.ddelta)[o] = from_f32<T>(dd);
      }
      if (m.start >> j & 1) {
        if (p.dstate0 && w.on) store_state<NP>(p.dstate0, q.seq(), p, w.d, dh);
        if (PACKED) q.prev((int)t - 1);
      }
    }
  }
  if (w.on) {
    float* pa = p.part_a + (int64_t)row * (p.N + 2) * p.D + w.d;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (i < p.N) pa[(int64_t)i * p.D] = dA[i];
    pa[(int64_t)p.N * p.D] = dD;
    pa[(int64_t)(p.N + 1) * p.D] = dbias;
  }
}

// dB and dC of every token: the sum of its tiles' partial rows, in the tiles' order
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_kernel(const float* part, T* dB, T* dC, int64_t rows_g, int N, int tiles) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t total = rows_g * 2 * N;
  if (i >= total) return;
  float s = 0.f;
  for (int k = 0; k < tiles; ++k) s += part[k * total + i];
  const int64_t r = i / (2 * N);
  const int c = (int)(i % (2 * N));
  if (c < N) dB[r * N + c] = from_f32<T>(s);
  else dC[r * N + c - N] = from_f32<T>(s);
}

// dA [D][N], dD [D], dbias [D] from the partial rows [parts][N + 2][D], in the parts' order
__global__ void __launch_bounds__(256) scan_params_kernel(const float* part, float* dA, float* dD, float* dbias,
                                                          int parts, int N, int D) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t total = (int64_t)(N + 2) * D;
  if (i >= total) return;
  float s = 0.f;
  for (int k = 0; k < parts; ++k) s += part[k * total + i];
  const int n = (int)(i / D), d = (int)(i % D);
  if (n < N) { if (dA) dA[(int64_t)d * N + n] = s; }
  else if (n == N) { if (dD) dD[d] = s; }
  else if (dbias) dbias[d] = s;
}

// One token per row: a lane owns one state of one channel at a time, a channel's states in neighbouring lanes, so that
// the state, nearly all of the traffic, is read and written in whole lines.
template <typename T>
__global__ void __launch_bounds__(256) scan_step_kernel(ScanArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t total = (int64_t)p.rows * p.D;
  if (i >= total) return;
  const int row = (int)(i / p.D), d = (int)(i % p.D), g = d / p.Dg;
  const float uu = to_f32(((const T*)p.u)[row * p.u_sb + d]);
  const float pre = to_f32(((const T*)p.delta)[row * p.delta_sb + d]) + (p.bias ? p.bias[d] : 0.f);
  const float dt = p.softplus ? softplus_hw(pre) : pre;
  const T* B = (const T*)p.B + row * p.B_sb + g * p.B_sg;
  const T* C = (const T*)p.C + row * p.C_sb + g * p.C_sg;
  float* h = p.state1 + i * p.N;
  float y = p.Dp ? p.Dp[d] * uu : 0.f;
  const float x = dt * uu;
  for (int n = 0; n < p.N; ++n) {
    const float v = fmaf(exp2_hw(dt * (p.A[(int64_t)d * p.N + n] * LOG2E_F)), h[n], x * to_f32(B[n]));
    h[n] = v;
    y = fmaf(to_f32(C[n]), v, y);
  }
  if (p.z) {
    const float zz = to_f32(((const T*)p.z)[row * p.z_sb + d]);
    y *= zz * sigmoid_hw(zz);
  }
  ((T*)p.out)[i] = from_f32<T>(y);
}

// ------------------------------------------------------------------------------------------------ host side
static int scan_check(const char* what, int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N, int64_t S,
                      const int32_t* offsets, int dtype) {
  DVAE_REQUIRE(dtype == DVAE_DT_F32 || dtype == DVAE_DT_BF16, "%s: dtype must be fp32 (0) or bf16 (1)", what);
  DVAE_REQUIRE(rows >= 0 && L >= 0 && D > 0 && G > 0 && D % G == 0, "%s: D must be a multiple of G", what);
  DVAE_REQUIRE(N > 0 && N <= SCAN_MAX_N, "%s: 1 to %d states per channel, got %ld", what, SCAN_MAX_N, (long)N);
  DVAE_REQUIRE(rows * L < (1ll << 31) && D < (1ll << 24) && rows < (1ll << 31), "%s: too large", what);
  DVAE_REQUIRE(!offsets || (rows == 1 && S >= 1 && S < (1ll << 30)), "%s: offsets go with one row and S >= 1", what);
  return 0;
}

static void scan_shape(ScanArgs& p, int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N, int64_t S) {
  p.rows = (int)rows; p.L = (int)L; p.D = (int)D; p.G = (int)G; p.N = (int)N; p.S = (int)S;
  p.Dg = (int)(D / G);
  p.tpg = (p.Dg + 63) / 64;
  p.ntiles = p.tpg * p.G;
  p.blocks = (int)ceil_div64(L, SCAN_Q);
}

// whether B and C of every token and group can be read as whole aligned words
static bool scan_words(const ScanArgs& p, int dtype, int NP) {
  if (p.N != NP) return false;
  if (dtype == DVAE_DT_F32) return true;
  const int64_t odd = p.B_sb | p.B_st | p.B_sg | p.C_sb | p.C_st | p.C_sg;
  return !(odd & 1) && !(((uintptr_t)p.B | (uintptr_t)p.C) & 3);
}

#define SCAN_LAUNCH(K, T, NP, grid, p, s)                                                             \
  do {                                                                                                \
    const bool fast__ = scan_words(p, sizeof(T) == 4 ? DVAE_DT_F32 : DVAE_DT_BF16, NP);               \
    if (p.offsets) {                                                                                  \
      if (fast__) DVAE_LAUNCH((K<T, NP, true, true>), dim3(grid), dim3(256), 0, s, p);                \
      else DVAE_LAUNCH((K<T, NP, true, false>), dim3(grid), dim3(256), 0, s, p);                      \
    } else {                                                                                          \
      if (fast__) DVAE_LAUNCH((K<T, NP, false, true>), dim3(grid), dim3(256), 0, s, p);               \
      else DVAE_LAUNCH((K<T, NP, false, false>), dim3(grid), dim3(256), 0, s, p);                     \
    }                                                                                                 \
  } while (0)
#define SCAN_DISPATCH(K, dtype, grid, p, s)                                                           \
  do {                                                                                                \
    if (dtype == DVAE_DT_F32) {                                                                       \
      if (p.N <= 8) SCAN_LAUNCH(K, float, 8, grid, p, s); else SCAN_LAUNCH(K, float, 16, grid, p, s); \
    } else {                                                                                          \
      if (p.N <= 8) SCAN_LAUNCH(K, bf16_t, 8, grid, p, s); else SCAN_LAUNCH(K, bf16_t, 16, grid, p, s); \
    }                                                                                                 \
  } while (0)

extern "C" int64_t dvae_selective_scan_ckpt_floats(int64_t rows, int64_t L, int64_t D, int64_t N) {
  return rows * ceil_div64(L, SCAN_Q) * N * D;
}

extern "C" int64_t dvae_selective_scan_bwd_ws_floats(int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N) {
  const int64_t tpg = ceil_div64(D / G, 64);
  return tpg * rows * L * G * 2 * N + rows * (N + 2) * D;
}

extern "C" int dvae_selective_scan_fwd(const void* u, int64_t u_sb, int64_t u_st, const void* delta, int64_t delta_sb,
                                       int64_t delta_st, const float* A, const void* B, int64_t B_sb, int64_t B_st,
                                       int64_t B_sg, const void* C, int64_t C_sb, int64_t C_st, int64_t C_sg,
                                       const float* Dp, const void* z, int64_t z_sb, int64_t z_st, const float* bias,
                                       int softplus, const float* state0, float* state1, const int32_t* offsets,
                                       void* out, float* ckpt, int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N,
                                       int64_t S, int dtype, dvae_stream_t stream) {
  const int rc = scan_check("selective_scan_fwd", rows, L, D, G, N, S, offsets, dtype);
  if (rc) return rc;
  if (rows * L == 0) return 0;
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.u_st = u_st; p.delta = delta; p.delta_sb = delta_sb; p.delta_st = delta_st; p.A = A;
  p.B = B; p.B_sb = B_sb; p.B_st = B_st; p.B_sg = B_sg; p.C = C; p.C_sb = C_sb; p.C_st = C_st; p.C_sg = C_sg;
  p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.z_st = z_st; p.bias = bias; p.softplus = softplus;
  p.state0 = state0; p.state1 = state1; p.offsets = offsets; p.out = out; p.ckpt = ckpt;
  scan_shape(p, rows, L, D, G, N, S);
  const int64_t grid = rows * ceil_div64(p.ntiles, 4);
  DVAE_REQUIRE(grid < (1ll << 31), "selective_scan_fwd: too many rows");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(rows * L * (double)e * ((z ? 4 : 3) * D + 2 * G * N), DVAE_UNIT_BYTE);
  SCAN_DISPATCH(scan_fwd_kernel, dtype, grid, p, ST(stream));
  DVAE_LAUNCH_CHECK("selective_scan_fwd");
  return 0;
}

extern "C" int dvae_selective_scan_bwd(const void* u, int64_t u_sb, int64_t u_st, const void* delta, int64_t delta_sb,
                                       int64_t delta_st, const float* A, const void* B, int64_t B_sb, int64_t B_st,
                                       int64_t B_sg, const void* C, int64_t C_sb, int64_t C_st, int64_t C_sg,
                                       const float* Dp, const void* z, int64_t z_sb, int64_t z_st, const float* bias,
                                       int softplus, const float* state0, const int32_t* offsets, const void* dout,
                                       int64_t dout_sb, int64_t dout_st, const float* dstate1, const float* ckpt,
                                       void* du, void* ddelta, float* dA, void* dB, void* dC, float* dD, void* dz,
                                       float* dbias, float* dstate0, int64_t rows, int64_t L, int64_t D, int64_t G,
                                       int64_t N, int64_t S, int dtype, float* ws, dvae_stream_t stream) {
  const int rc = scan_check("selective_scan_bwd", rows, L, D, G, N, S, offsets, dtype);
  if (rc) return rc;
  DVAE_REQUIRE(rows * L > 0, "selective_scan_bwd: no tokens");
  DVAE_REQUIRE(!z || dz, "selective_scan_bwd: dz is needed with z");
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.u_st = u_st; p.delta = delta; p.delta_sb = delta_sb; p.delta_st = delta_st; p.A = A;
  p.B = B; p.B_sb = B_sb; p.B_st = B_st; p.B_sg = B_sg; p.C = C; p.C_sb = C_sb; p.C_st = C_st; p.C_sg = C_sg;
  p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.z_st = z_st; p.bias = bias; p.softplus = softplus;
  p.state0 = state0; p.offsets = offsets; p.dout = dout; p.dout_sb = dout_sb; p.dout_st = dout_st;
  p.dstate1 = dstate1; p.dstate0 = dstate0; p.ckpt = const_cast<float*>(ckpt);
  p.du = du; p.ddelta = ddelta; p.dz = dz;
  scan_shape(p, rows, L, D, G, N, S);
  p.part_bc = ws;
  p.part_a = ws + (int64_t)p.tpg * rows * L * G * 2 * N;
  const int64_t grid = rows * ceil_div64(p.ntiles, 4);
  DVAE_REQUIRE(grid < (1ll << 31), "selective_scan_bwd: too many rows");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(rows * L * (double)e * ((z ? 7 : 5) * D + 4 * G * N), DVAE_UNIT_BYTE);
  SCAN_DISPATCH(scan_bwd_kernel, dtype, grid, p, ST(stream));
  DVAE_LAUNCH_CHECK("selective_scan_bwd");
  const int64_t bc = rows * L * G;
  const dim3 gbc((unsigned)ceil_div64(bc * 2 * N, 256));
  if (dtype == DVAE_DT_F32)
    DVAE_LAUNCH((scan_bc_kernel<float>), gbc, dim3(256), 0, ST(stream), p.part_bc, (float*)dB, (float*)dC, bc, p.N, p.tpg);
  else
    DVAE_LAUNCH((scan_bc_kernel<bf16_t>), gbc, dim3(256), 0, ST(stream), p.part_bc, (bf16_t*)dB, (bf16_t*)dC, bc, p.N, p.tpg);
  DVAE_LAUNCH(scan_params_kernel, dim3((unsigned)ceil_div64((int64_t)(p.N + 2) * D, 256)), dim3(256), 0, ST(stream),
              p.part_a, dA, dD, dbias, p.rows, p.N, p.D);
  DVAE_LAUNCH_CHECK("selective_scan_bwd: sums");
  return 0;
}

extern "C" int dvae_selective_scan_step(float* state, const void* u, int64_t u_sb, const void* delta, int64_t delta_sb,
                                        const float* A, const void* B, int64_t B_sb, int64_t B_sg, const void* C,
                                        int64_t C_sb, int64_t C_sg, const float* Dp, const void* z, int64_t z_sb,
                                        const float* bias, int softplus, void* out, int64_t rows, int64_t D, int64_t G,
                                        int64_t N, int dtype, dvae_stream_t stream) {
  const int rc = scan_check("selective_scan_step", rows, 1, D, G, N, rows, nullptr, dtype);
  if (rc) return rc;
  if (rows == 0) return 0;
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.delta = delta; p.delta_sb = delta_sb; p.A = A; p.B = B; p.B_sb = B_sb; p.B_sg = B_sg;
  p.C = C; p.C_sb = C_sb; p.C_sg = C_sg; p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.bias = bias; p.softplus = softplus;
  p.state1 = state; p.out = out;
  scan_shape(p, rows, 1, D, G, N, rows);
  const int64_t grid = ceil_div64(rows * D, 256);
  DVAE_REQUIRE(grid < (1ll << 31), "selective_scan_step: too many rows");
  DVAE_WORK(rows * (double)D * N * 8, DVAE_UNIT_BYTE);
  if (dtype == DVAE_DT_F32) DVAE_LAUNCH((scan_step_kernel<float>), dim3(grid), dim3(256), 0, ST(stream), p);
  else DVAE_LAUNCH((scan_step_kernel<bf16_t>), dim3(grid), dim3(256), 0, ST(stream), p);
  DVAE_LAUNCH_CHECK("selective_scan_step");
  return 0;
}
