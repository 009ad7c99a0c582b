// The short causal convolution over time, depthwise and channels-last: out[t] = act(bias + sum_k w[k] x[t - (W-1) + k]),
// where tokens before a sequence's first are the carried state, or zero.  Bound by memory: every element of x is read
// once (and a block's first W - 1 rows twice, out of the L2) and kept in registers for the W outputs that use it.
//
// A lane owns one 32-bit word of a row (V = 2 bf16 channels where the tensors' alignment allows it, else one): with 16
// bytes per lane the window, the taps and what is in flight take so many registers that too few waves run (backward, 8 x
// 2048 x 2048 bf16, four taps: 125 us with 16 bytes, 72 with 8, 57 with 4).  A wave takes p.tb consecutive tokens.
// CONV_AHEAD tokens are in flight at any time: a token's registers receive the one CONV_AHEAD further on as soon as it has
// been used.  A batch is walked as one line of tokens, sequence after sequence, so short clips fill the chip like long
// sequences do.
//
// 8 x 2048 x 2048 bf16, four taps: forward 33 us (4.1 TB/s of x and out), backward 57 us (3.5 TB/s of x, dout and dx) and
// 4 us for the sums of its partial rows; 32 x 1024 fp32, one token: 2.7 us.
#include "seq_common.h"

#define CONV_AHEAD 8

struct ConvArgs {
  const void *x, *dout, *state0, *dstate1;
  int64_t x_sb, x_st, dout_sb, dout_st;
  const float *w, *bias;
  void *out, *state1, *dx, *dstate0;
  float* part;                 // [workgroup row][W + 1][D]: partial sums of dw and dbias
  const int32_t* offsets;
  int D, S, L, tokens, silu, tiles;
  int tb;                      // tokens whose inputs a wave reads
};

// where token t of the walk's sequence lies
template <typename T>
__device__ __forceinline__ const T* token(const void* base, const SeqWalk& q, int64_t sb, int64_t st, int t) {
  return (const T*)base + (q.off ? t * st : q.s * sb + (t - q.b) * st);
}

// The rows of a tensor token by token, in the order of the walk, CONV_AHEAD of them requested; the last one again when
// there are no more.
template <typename T, int V> struct Feed {
  const T* p;                  // row of the next token to be requested
  int64_t st, turn;            // to the next token's row, within a sequence of the batch and into the next one
  int left, L, more;           // tokens left in the sequence (batch) and of those to be requested
  Packed<T, V> raw[CONV_AHEAD];
  __device__ __forceinline__ Feed(const void* base, const SeqWalk& q, int64_t sb, int64_t st_, int t0, int n, int d)
      : st(st_), turn(st_), left(q.tokens), L(q.tokens), more(n - 1) {
    p = (const T*)base + t0 * st;
    if (!q.off) {
      L = q.L;
      p = (const T*)base + q.s * sb + (t0 - q.b) * st;
      turn = sb - (int64_t)(L - 1) * st;
      left = q.e - t0;
    }
#pragma unroll
    for (int j = 0; j < CONV_AHEAD; ++j) request(j, d);
  }
  __device__ __forceinline__ void request(int j, int d) {
    raw[j].load(p + d);
    if (more > 0) {
      --more;
      --left;
      p += left ? st : turn;
      left = left ? left : L;
    }
  }
  // token j of the group; its place is taken by the one CONV_AHEAD further on
  __device__ __forceinline__ void take(int j, int d, float (&v)[V]) {
    raw[j].get(v);
    request(j, d);
  }
};

// the input at position t of the walk's sequence, t >= b - (W-1): a token, or what was carried in
template <typename T, int V, int W>
__device__ __forceinline__ void load_input(const ConvArgs& p, const SeqWalk& q, int t, int d, float (&v)[V]) {
  if (t >= q.b) load_pack<T, V>(token<T>(p.x, q, p.x_sb, p.x_st, t) + d, v);
  else if (p.state0) load_pack<T, V>((const T*)p.state0 + ((int64_t)q.s * (W - 1) + (t - q.b + W - 1)) * p.D + d, v);
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
  }
}

template <int V, int W>
__device__ __forceinline__ void load_weights(const ConvArgs& p, int d, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = p.bias ? p.bias[d + i] : 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][i] = p.w[(int64_t)(d + i) * W + k];
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(256) conv_fwd_kernel(ConvArgs p) {
  const int d = ((int)(blockIdx.x % p.tiles) * 64 + (threadIdx.x & 63)) * V;
  const int t0 = ((int)(blockIdx.x / p.tiles) * 4 + uniform(threadIdx.x >> 6)) * p.tb;
  if (t0 >= p.tokens) return;
  const int t1 = min(t0 + p.tb, p.tokens);
  float w[W][V], bias[V], win[W][V];
  load_weights<V, W>(p, d < p.D ? d : 0, w, bias);
  SeqWalk q = {p.offsets, p.S, p.L, p.tokens, 0, 0, 0};
  q.seek(t0);
  if (p.state1 && p.offsets) {                 // sequences without tokens end with what they entered with
    q.for_empty(t0 / p.tb, (p.tokens + p.tb - 1) / p.tb, [&](int s) {
      if (d >= p.D) return;
#pragma unroll
      for (int k = 0; k + 1 < W; ++k) {
        float v[V] = {};
        const int64_t i = ((int64_t)s * (W - 1) + k) * p.D + d;
        if (p.state0) load_pack<T, V>((const T*)p.state0 + i, v);
        store_pack<T, V>((T*)p.state1 + i, v);
      }
    });
  }
  if (d >= p.D) return;
  if (q.s < q.S && q.b < t0) {
#pragma unroll
    for (int k = 1; k < W; ++k) load_input<T, V, W>(p, q, t0 - W + k, d, win[k]);
  }
  T* out = (T*)p.out + d;
  Feed<T, V> x(p.x, q, p.x_sb, p.x_st, t0, t1 - t0, d);
  for (int g = t0; g < t1; g += CONV_AHEAD) {
#pragma unroll
    for (int j = 0; j < CONV_AHEAD; ++j) {
      const int t = g + j;
      if (t >= t1) continue;
      float y[V], now[V];
      x.take(j, d, now);
      if (q.s >= q.S || t < q.b) {
        const float zero[V] = {};
        store_pack<T, V>(out + (int64_t)t * p.D, zero);
        continue;
      }
      if (t == q.b) {
#pragma unroll
        for (int k = 1; k < W; ++k) load_input<T, V, W>(p, q, t - W + k, d, win[k]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) win[k][i] = win[k + 1][i];
        win[W - 1][i] = now[i];
        y[i] = bias[i];
#pragma unroll
        for (int k = 0; k < W; ++k) y[i] = fmaf(w[k][i], win[k][i], y[i]);
        if (p.silu) y[i] *= sigmoid_hw(y[i]);
      }
      store_pack<T, V>(out + (int64_t)t * p.D, y);
      if (t + 1 == q.e) {
        if (p.state1) {
#pragma unroll
          for (int k = 1; k < W; ++k)
            store_pack<T, V>((T*)p.state1 + ((int64_t)q.s * (W - 1) + k - 1) * p.D + d, win[k]);
        }
        q.next(t + 1);
      }
    }
  }
}

// gradient of the value before the activation at token t of the walk's sequence; the window ends up in win
template <typename T, int V, int W>
__device__ __forceinline__ void grad_pre(const ConvArgs& p, const float (&w)[W][V], const float (&bias)[V],
                                         const float (&win)[W][V], const float (&g)[V], float (&dp)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    dp[i] = g[i];
    if (p.silu) {
      float y = bias[i];
#pragma unroll
      for (int k = 0; k < W; ++k) y = fmaf(w[k][i], win[k][i], y);
      const float s = sigmoid_hw(y);
      dp[i] *= s * fmaf(y, 1.f - s, 1.f);
    }
  }
}

// dx[t] = sum_k w[k] dpre[t + (W-1) - k] over the tokens of the same sequence; dw[k] = sum_t dpre[t] x[t - (W-1) + k].
// A wave's own tokens are p.tb - (W-1); it runs W - 1 past them, whose dpre its last ones need.
template <typename T, int V, int W>
__global__ void __launch_bounds__(256) conv_bwd_kernel(ConvArgs p) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int d0 = ((int)(blockIdx.x % p.tiles) * 64 + lane) * V;
  const bool on = d0 < p.D;
  const int d = on ? d0 : 0;
  const int t0 = ((int)(blockIdx.x / p.tiles) * 4 + wave) * (p.tb - (W - 1));
  const int t1 = min(t0 + p.tb - (W - 1), p.tokens);
  float w[W][V], bias[V], win[W][V] = {}, acc[W][V] = {}, dw[W][V] = {}, db[V] = {};
  if (t0 < p.tokens) {
    load_weights<V, W>(p, d, w, bias);
    SeqWalk q = {p.offsets, p.S, p.L, p.tokens, 0, 0, 0};
    q.seek(t0);
    if (q.s < q.S && q.b < t0) {
#pragma unroll
      for (int k = 1; k < W; ++k) load_input<T, V, W>(p, q, t0 - W + k, d, win[k]);
    }
    const int n = min(t1 + W - 1, p.tokens) - t0;
    Feed<T, V> x(p.x, q, p.x_sb, p.x_st, t0, n, d), go(p.dout, q, p.dout_sb, p.dout_st, t0, n, d);
    for (int g0 = t0; g0 < t1 + W - 1; g0 += CONV_AHEAD) {
#pragma unroll
      for (int j = 0; j < CONV_AHEAD; ++j) {
        const int t = g0 + j;
        if (t >= t1 + W - 1) continue;
        float now[V], g[V], dp[V];
        x.take(j, d, now);
        go.take(j, d, g);
        if (t < p.tokens && q.s < q.S && t >= q.b) {
          if (t == q.b) {
#pragma unroll
            for (int k = 1; k < W; ++k) load_input<T, V, W>(p, q, t - W + k, d, win[k]);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int k = 0; k + 1 < W; ++k) win[k][i] = win[k + 1][i];
            win[W - 1][i] = now[i];
          }
          grad_pre<T, V, W>(p, w, bias, win, g, dp);
#pragma unroll
          for (int k = 0; k < W; ++k)
            if (t - (W - 1) + k >= q.b) {
#pragma unroll
              for (int i = 0; i < V; ++i) acc[k][i] = fmaf(w[k][i], dp[i], acc[k][i]);
            }
          if (p.dstate1 && t >= q.e - (W - 1)) {
            float c[V];
            load_pack<T, V>((const T*)p.dstate1 + ((int64_t)q.s * (W - 1) + t - q.e + W - 1) * p.D + d, c);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[W - 1][i] += c[i];
          }
          if (t < t1) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              db[i] += dp[i];
#pragma unroll
              for (int k = 0; k < W; ++k) dw[k][i] = fmaf(dp[i], win[k][i], dw[k][i]);
            }
          }
          if (t + 1 == q.e) q.next(t + 1);
        }
        if (t - (W - 1) >= t0 && on) store_pack<T, V>((T*)p.dx + (int64_t)(t - (W - 1)) * p.D + d, acc[0]);
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) acc[k][i] = k + 1 < W ? acc[k + 1 < W ? k + 1 : k][i] : 0.f;
      }
    }
  }
  __shared__ float red[3][(W + 1) * V][64];
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int k = 0; k < W; ++k) red[wave - 1][k * V + i][lane] = dw[k][i];
      red[wave - 1][W * V + i][lane] = db[i];
    }
  }
  __syncthreads();
  if (wave == 0 && on) {
    float* q = p.part + (int64_t)(blockIdx.x / p.tiles) * (W + 1) * p.D + d;
#pragma unroll
    for (int k = 0; k <= W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = k < W ? dw[k < W ? k : 0][i] : db[i];
        for (int o = 0; o < 3; ++o) s += red[o][k * V + i][lane];
        q[(int64_t)k * p.D + i] = s;
      }
  }
}

// dw [D][W] and dbias [D] from the partial rows [parts][W + 1][D]
__global__ void __launch_bounds__(64 * SUM_WAVES) conv_params_kernel(const float* part, float* dw, float* dbias, int parts,
                                                                     int W, int D) {
  const int64_t total = (int64_t)(W + 1) * D;
  const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float s = column_sum(part, parts, total, i, i < total);
  if (threadIdx.x >= 64 || i >= total) return;
  const int k = (int)(i / D), d = (int)(i % D);
  if (k < W) { if (dw) dw[(int64_t)d * W + k] = s; }
  else if (dbias) dbias[d] = s;
}

// the gradient of the carried inputs: row j of a sequence's state reaches the tokens p <= j with tap j - p, and the
// final state where the sequence is shorter than the window, or has no tokens
template <typename T, int W>
__global__ void __launch_bounds__(256) conv_dstate_kernel(ConvArgs p) {
  const int d = (int)(blockIdx.x % p.tiles) * 256 + threadIdx.x;
  SeqWalk q = {p.offsets, p.S, p.L, p.tokens, (int)(blockIdx.x / p.tiles), 0, 0};
  q.load();
  if (d >= p.D) return;
  float w[W][1], bias[1], ds[W] = {};
  load_weights<1, W>(p, d, w, bias);
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    if (q.b + j >= q.e) continue;
    float win[W][1], g[1], dp[1];
#pragma unroll
    for (int k = 0; k < W; ++k) load_input<T, 1, W>(p, q, q.b + j - (W - 1) + k, d, win[k]);
    load_pack<T, 1>(token<T>(p.dout, q, p.dout_sb, p.dout_st, q.b + j) + d, g);
    grad_pre<T, 1, W>(p, w, bias, win, g, dp);
#pragma unroll
    for (int r = j; r < W - 1; ++r) ds[r] = fmaf(w[r - j][0], dp[0], ds[r]);
  }
#pragma unroll
  for (int r = 0; r < W - 1; ++r) {
    const int from = r - max(q.e - q.b, 0);
    if (p.dstate1 && from >= 0) ds[r] += to_f32(((const T*)p.dstate1)[((int64_t)q.s * (W - 1) + from) * p.D + d]);
    ((T*)p.dstate0)[((int64_t)q.s * (W - 1) + r) * p.D + d] = from_f32<T>(ds[r]);
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(256) conv_step_kernel(ConvArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = p.D / V;
  if (i >= (int64_t)p.tokens * per) return;
  const int row = (int)(i / per), d = (int)(i % per) * V;
  float w[W][V], bias[V], win[W][V], y[V];
  load_weights<V, W>(p, d, w, bias);
  T* st = (T*)p.state1 + (int64_t)row * (W - 1) * p.D + d;
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) load_pack<T, V>(st + (int64_t)k * p.D, win[k]);
  load_pack<T, V>((const T*)p.x + row * p.x_sb + d, win[W - 1]);
#pragma unroll
  for (int i2 = 0; i2 < V; ++i2) {
    y[i2] = bias[i2];
#pragma unroll
    for (int k = 0; k < W; ++k) y[i2] = fmaf(w[k][i2], win[k][i2], y[i2]);
    if (p.silu) y[i2] *= sigmoid_hw(y[i2]);
  }
  store_pack<T, V>((T*)p.out + (int64_t)row * p.D + d, y);
#pragma unroll
  for (int k = 0; k + 1 < W; ++k) store_pack<T, V>(st + (int64_t)k * p.D, win[k + 1]);
}

// ------------------------------------------------------------------------------------------------ host side
static int conv_check(const char* what, int64_t rows, int64_t L, int64_t D, int64_t W, int64_t S,
                      const int32_t* offsets, int dtype) {
  DVAE_REQUIRE(dtype == DVAE_DT_F32 || dtype == DVAE_DT_BF16, "%s: dtype must be fp32 (0) or bf16 (1)", what);
  DVAE_REQUIRE(W >= 2 && W <= 4, "%s: 2 to 4 taps, got %ld", what, (long)W);
  DVAE_REQUIRE(rows >= 0 && L >= 0 && D > 0 && D < (1ll << 24), "%s: bad shape", what);
  DVAE_REQUIRE(rows < (1ll << 31) && L < (1ll << 31) && rows * L < SEQ_MAX_TOKENS, "%s: too many tokens", what);
  DVAE_REQUIRE(!offsets || (rows == 1 && S >= 1 && S < (1ll << 30)), "%s: offsets go with one row and S >= 1", what);
  return 0;
}

// two bf16 channels per lane where every row of every tensor starts on 4 bytes
static bool conv_pairs(int64_t D, int dtype, const void* a, int64_t a_sb, int64_t a_st, const void* b, int64_t b_sb,
                       int64_t b_st, const void* c, const void* d, const void* e) {
  const uintptr_t ptrs = (uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d | (uintptr_t)e;
  return dtype == DVAE_DT_BF16 && !(ptrs & 3) && !((D | a_sb | a_st | b_sb | b_st) & 1);
}

// Tokens per wave: 32, or fewer (at least `least`) where that would leave less than four waves per SIMD: 5003 x 1001 fp32
// forward, three taps: 18.4 us with 32, 14.6 with 16; 8 x 2048 x 2048 bf16: 32 with 32, 35 with 16, 39 with 64.
// `past`: tokens that a wave reads beyond its own.
static int conv_tb(int64_t tokens, int64_t tiles, int past, int least) {
  int tb = 32;
  while (tb > least && tiles * ceil_div64(tokens, tb - past) < 4096) tb /= 2;
  return tb;
}
static int64_t conv_parts(int64_t tokens, int64_t D, int v, int W) {
  return ceil_div64(tokens, 4 * (conv_tb(tokens, ceil_div64(D, 64 * v), W - 1, 16) - (W - 1)));
}

#define CONV_W(K, T, V, W, grid, p, s)                                                     \
  do {                                                                                     \
    if (W == 2) DVAE_LAUNCH((K<T, V, 2>), grid, dim3(256), 0, s, p);                       \
    else if (W == 3) DVAE_LAUNCH((K<T, V, 3>), grid, dim3(256), 0, s, p);                  \
    else DVAE_LAUNCH((K<T, V, 4>), grid, dim3(256), 0, s, p);                              \
  } while (0)
#define CONV_DISPATCH(K, dtype, pairs, W, grid, p, s)                                      \
  do {                                                                                     \
    if (dtype == DVAE_DT_F32) {                                                            \
      CONV_W(K, float, 1, W, grid, p, s);                                                  \
    } else {                                                                               \
      if (pairs) CONV_W(K, bf16_t, 2, W, grid, p, s); else CONV_W(K, bf16_t, 1, W, grid, p, s); \
    }                                                                                      \
  } while (0)


extern "C" int dvae_short_conv_fwd(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias, int silu,
                                   const void* state0, void* state1, const int32_t* offsets, void* out, int64_t rows,
                                   int64_t L, int64_t D, int64_t W, int64_t S, int dtype, dvae_stream_t stream) {
  const int rc = conv_check("short_conv_fwd", rows, L, D, W, S, offsets, dtype);
  if (rc) return rc;
  if (rows * L == 0) return 0;
  ConvArgs p = {};
  p.x = x; p.x_sb = x_sb; p.x_st = x_st; p.w = w; p.bias = bias; p.silu = silu; p.state0 = state0; p.state1 = state1;
  p.offsets = offsets; p.out = out; p.D = (int)D; p.S = (int)(offsets ? S : rows); p.L = (int)L;
  p.tokens = (int)(rows * L);
  const bool pairs = conv_pairs(D, dtype, x, x_sb, x_st, nullptr, 0, 0, state0, state1, out);
  p.tiles = (int)ceil_div64(D, 64 * (pairs ? 2 : 1));
  p.tb = conv_tb(p.tokens, p.tiles, 0, 8);
  const int64_t grid = p.tiles * ceil_div64(p.tokens, 4 * p.tb);
  DVAE_REQUIRE(launch_fits(grid, 256), "short_conv_fwd: too large for one launch");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(2.0 * p.tokens * D * e, DVAE_UNIT_BYTE);
  CONV_DISPATCH(conv_fwd_kernel, dtype, pairs, W, dim3((unsigned)grid), p, ST(stream));
  DVAE_LAUNCH_CHECK("short_conv_fwd");
  return 0;
}

extern "C" int64_t dvae_short_conv_bwd_ws_floats(int64_t rows, int64_t L, int64_t D, int64_t W) {
  if (rows * L <= 0 || W < 2 || W > 4) return 0;
  const int64_t a = conv_parts(rows * L, D, 1, (int)W), b = conv_parts(rows * L, D, 2, (int)W);
  return (a > b ? a : b) * (W + 1) * D;
}

extern "C" int dvae_short_conv_bwd(const void* x, int64_t x_sb, int64_t x_st, const float* w, const float* bias, int silu,
                                   const void* state0, const int32_t* offsets, const void* dout, int64_t dout_sb,
                                   int64_t dout_st, const void* dstate1, void* dx, float* dw, float* dbias,
                                   void* dstate0, int64_t rows, int64_t L, int64_t D, int64_t W, int64_t S, int dtype,
                                   float* ws, dvae_stream_t stream) {
  const int rc = conv_check("short_conv_bwd", rows, L, D, W, S, offsets, dtype);
  if (rc) return rc;
  DVAE_REQUIRE(rows * L > 0, "short_conv_bwd: no tokens");
  ConvArgs p = {};
  p.x = x; p.x_sb = x_sb; p.x_st = x_st; p.w = w; p.bias = bias; p.silu = silu; p.state0 = state0; p.offsets = offsets;
  p.dout = dout; p.dout_sb = dout_sb; p.dout_st = dout_st; p.dstate1 = dstate1; p.dx = dx; p.dstate0 = dstate0;
  p.D = (int)D; p.S = (int)(offsets ? S : rows); p.L = (int)L; p.tokens = (int)(rows * L); p.part = ws;
  const bool pairs = conv_pairs(D, dtype, x, x_sb, x_st, dout, dout_sb, dout_st, state0, dstate1, dx);
  p.tiles = (int)ceil_div64(D, 64 * (pairs ? 2 : 1));
  p.tb = conv_tb(p.tokens, p.tiles, (int)W - 1, 16);
  const int64_t parts = conv_parts(p.tokens, D, pairs ? 2 : 1, (int)W);
  DVAE_REQUIRE(launch_fits(p.tiles * parts, 256) && (!dstate0 || launch_fits(ceil_div64(D, 256) * p.S, 256)),
               "short_conv_bwd: too large for one launch");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(3.0 * p.tokens * D * e, DVAE_UNIT_BYTE);
  CONV_DISPATCH(conv_bwd_kernel, dtype, pairs, W, dim3((unsigned)(p.tiles * parts)), p, ST(stream));
  DVAE_LAUNCH_CHECK("short_conv_bwd");
  DVAE_LAUNCH(conv_params_kernel, dim3((unsigned)ceil_div64((W + 1) * D, 64)), dim3(64 * SUM_WAVES), 0, ST(stream), ws, dw,
              dbias, (int)parts, (int)W, (int)D);
  if (dstate0) {
    p.tiles = (int)ceil_div64(D, 256);
    const dim3 grid((unsigned)(p.tiles * p.S));
#define CONV_DSTATE(T)                                                                     \
  do {                                                                                     \
    if (W == 2) DVAE_LAUNCH((conv_dstate_kernel<T, 2>), grid, dim3(256), 0, ST(stream), p); \
    else if (W == 3) DVAE_LAUNCH((conv_dstate_kernel<T, 3>), grid, dim3(256), 0, ST(stream), p); \
    else DVAE_LAUNCH((conv_dstate_kernel<T, 4>), grid, dim3(256), 0, ST(stream), p);       \
  } while (0)
    if (dtype == DVAE_DT_F32) CONV_DSTATE(float); else CONV_DSTATE(bf16_t);
  }
  DVAE_LAUNCH_CHECK("short_conv_bwd: sums");
  return 0;
}

extern "C" int dvae_short_conv_step(void* state, const void* x, int64_t x_sb, const float* w, const float* bias, int silu,
                                    void* out, int64_t rows, int64_t D, int64_t W, int dtype, dvae_stream_t stream) {
  const int rc = conv_check("short_conv_step", rows, 1, D, W, rows, nullptr, dtype);
  if (rc) return rc;
  if (rows == 0) return 0;
  ConvArgs p = {};
  p.x = x; p.x_sb = x_sb; p.w = w; p.bias = bias; p.silu = silu; p.state1 = state; p.out = out; p.D = (int)D;
  p.tokens = (int)rows;
  const bool pairs = conv_pairs(D, dtype, x, x_sb, 0, nullptr, 0, 0, state, out, nullptr);
  const int64_t grid = ceil_div64(rows * (D / (pairs ? 2 : 1)), 256);
  DVAE_REQUIRE(launch_fits(grid, 256), "short_conv_step: too large for one launch");
  DVAE_WORK((2.0 * W) * rows * D * (dtype == DVAE_DT_F32 ? 4 : 2), DVAE_UNIT_BYTE);
  CONV_DISPATCH(conv_step_kernel, dtype, pairs, W, dim3((unsigned)grid), p, ST(stream));
  DVAE_LAUNCH_CHECK("short_conv_step");
  return 0;
}
