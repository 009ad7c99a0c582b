// The selective state-space scan, channels-last.  Per channel d with N states, token by token within a sequence:
//   dt    = softplus(delta + bias)                       (softplus optional)
//   h[n]  = exp(dt A[d,n]) h[n] + dt u B[n]              B, C shared by the channels of a group
//   out   = (sum_n C[n] h[n] + D u) * silu(z)            D and z optional
// States, step sizes and sums are fp32 whatever the activations' type; the output is rounded once.
//
// A lane owns one channel and keeps its N states in registers, so the sum over n is a chain of fused multiply-adds and
// neighbouring lanes read neighbouring channels.  B and C of a token are the same for all lanes: they come through the
// scalar unit and enter the vector instructions as scalar operands.
//
// One wave per 64 channels of a sequence would leave most of the chip idle where there are few sequences, so the time
// axis is split into chunks that run side by side.  A chunk needs the state that enters it: a first pass computes each
// chunk's state as if it started from zero (and the sum of its step sizes, whose exponential is the chunk's decay), a
// second joins those along the axis, the third computes the outputs.  The way back does the same from the right.  Both
// extra passes are left out where there is one chunk.
#include "seq_common.h"

#define SCAN_Q 8       // tokens per block: what is loaded ahead, and how far apart training keeps states
#define SCAN_MAX_N 16
#define SCAN_WAVES 2048    // two waves for each of the chip's SIMDs

struct ScanArgs {
  const void *u, *delta, *z, *B, *C, *dout;
  int64_t u_sb, u_st, delta_sb, delta_st, z_sb, z_st, B_sb, B_st, B_sg, C_sb, C_st, C_sg, dout_sb, dout_st;
  const float *A, *Dp, *bias, *state0;
  const float* dstate1;
  float *state1, *dstate0;
  void *out, *du, *ddelta, *dz;
  float *ckpt;                 // [row][block of SCAN_Q tokens][n][D]: the state that enters the block
  float *part_bc, *part_a;     // partial sums of the gradients of B and C, and of A, D and bias
  float *enter, *leave;        // the states that enter the chunks, and the adjoints that enter them from the right
  float *sumdt, *keep;         // [row][chunk][D]: sum of step sizes; [row][chunk]: 1 where no sequence starts
  const int32_t* offsets;
  int rows, L, D, G, N, S, Dg, tpg, wpg, softplus, blocks;    // tpg: tiles of 64 channels per group
  int nch, CL, enter_row, enter_step;   // chunks, their tokens; slots of `enter` per row and from chunk to chunk
};

// A as the kernels use it, in powers of two.  An infinite one becomes the largest finite number: a step size of 0, which
// stands for tokens that are not there, has to leave the state as it is.
__device__ __forceinline__ float decay_rate(float a) {
  a *= LOG2E_F;
  return fabsf(a) > 3.402823466e38f ? copysignf(3.402823466e38f, a) : a;
}

// what happens inside a block of n tokens from t0 on: bit j of `start` / `end` / `valid`: token t0 + j is its
// sequence's first / its sequence's last / in a sequence at all
struct Marks { uint32_t start, end, valid; };

__device__ __forceinline__ Marks block_marks(SeqWalk w, int t0, int n) {
  Marks m = {0u, 0u, 0u};
  const uint32_t all = (1u << n) - 1u;
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

// The N values of B or C at one token, element by element: other numbers of states than 8 and 16, and bf16 rows off 4 bytes.
// No scalar loads of 16 bits exist, so in bf16 these come through the vector unit, the same for all lanes: 8 x 2048 x 2048
// with 12 states 541 us for the outputs and 1388 for the way back, with 16 states 156 and 496.
template <typename T, int NP> __device__ __forceinline__ void load_each(const T* p, int N, float (&v)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; ++n) v[n] = n < N ? to_f32(p[n]) : 0.f;
}

// B and C, requested a token ahead.  FAST: N == NP and 4-byte aligned, read as whole words.  Scalar loads return in any
// order, so waiting for one means waiting for all: `arrived` makes the words of this token a dependence of the address of
// the next one's, which puts the wait before the next request and a token's arithmetic between a request and its wait.
template <int K> struct Words { typedef uint32_t vec __attribute__((ext_vector_type(K), aligned(4))); };
template <typename T, int NP, bool FAST> struct BCAhead {
  typename Words<NP * sizeof(T) / 4>::vec b, c;
  typedef typename Words<NP * sizeof(T) / 4>::vec vec;
  __device__ __forceinline__ void request(const T* B, const T* C, int) {
    b = *(const DVAE_UNIFORM vec*)(uint64_t)B;
    c = *(const DVAE_UNIFORM vec*)(uint64_t)C;
  }
  __device__ __forceinline__ void request_b(const T* B, int) { b = *(const DVAE_UNIFORM vec*)(uint64_t)B; }
  __device__ __forceinline__ void arrived(const T*& B, const T*& C) {
    asm volatile("" : "+s"(b), "+s"(c), "+s"(B), "+s"(C));
  }
  __device__ __forceinline__ void arrived_b(const T*& B) { asm volatile("" : "+s"(b), "+s"(B)); }
  // (alone, C travels in b's place: request_b, arrived_b and get_b serve either)
  static __device__ __forceinline__ void unpack(const vec w, float (&v)[NP]) {
#pragma unroll
    for (int n = 0; n < NP; ++n)
      v[n] = sizeof(T) == 4 ? __uint_as_float(w[n * sizeof(T) / 4])
                            : __uint_as_float(n & 1 ? w[n / 2] & 0xffff0000u : w[n / 2] << 16);
  }
  __device__ __forceinline__ void get(float (&bv)[NP], float (&cv)[NP]) const { unpack(b, bv); unpack(c, cv); }
  __device__ __forceinline__ void get_b(float (&bv)[NP]) const { unpack(b, bv); }
};
template <typename T, int NP> struct BCAhead<T, NP, false> {
  float b[NP], c[NP];
  __device__ __forceinline__ void request(const T* B, const T* C, int N) {
    load_each(B, N, b);
    load_each(C, N, c);
  }
  __device__ __forceinline__ void request_b(const T* B, int N) { load_each(B, N, b); }
  __device__ __forceinline__ void arrived(const T*&, const T*&) {}
  __device__ __forceinline__ void arrived_b(const T*&) {}
  __device__ __forceinline__ void get(float (&bv)[NP], float (&cv)[NP]) const {
#pragma unroll
    for (int n = 0; n < NP; ++n) { bv[n] = b[n]; cv[n] = c[n]; }
  }
  __device__ __forceinline__ void get_b(float (&bv)[NP]) const {
#pragma unroll
    for (int n = 0; n < NP; ++n) bv[n] = b[n];
  }
};

// Asks for one element of each end of B's and C's rows of a block of n tokens (four lanes alike), so that the lines are in
// the L2 when the scalar unit asks for them a token ahead: from there that is time enough, from memory it is not.  Measured
// with and without: 8 x 2048 x 2048 backward fp32 610 and 640 us, bf16 565 and 574; outputs of 1 x 4096 45 and 48 us.  The
// chunk passes read one of the two only and lose by it: 8 x 2048 x 2048 fp32, adjoints 153 and 140 us.
template <typename T>
__device__ __forceinline__ T touch_rows(const T* B, int64_t b_st, const T* C, int64_t c_st, int n, int N, int lane) {
  const int j = min(lane & 7, n - 1);
  return (lane & 8 ? C + j * c_st : B + j * b_st)[lane & 16 ? N - 1 : 0];
}
__device__ __forceinline__ void touched(float v) { asm volatile("" :: "v"(v)); }
__device__ __forceinline__ void touched(bf16_t v) { asm volatile("" :: "v"((uint32_t)v)); }

// 64 channels of one group, one chunk of one row (of narrower groups the lanes left over repeat the last channel: 8 x 2048 x
// 2048 bf16 in 64 groups of 32, outputs 366 us and way back 1666, in one group 156 and 496).  A workgroup's tiles are
// neighbours in a group; a tile is the work of one wave, or of `share` waves that have a part of the states each.
struct Tile {
  int g, d, lane, wave, part, chunk, row, t0, t1;
  bool on, idle;
  __device__ __forceinline__ explicit Tile(const ScanArgs& p, int tiles = 4, int share = 1) {
    lane = threadIdx.x & 63;
    wave = uniform(threadIdx.x >> 6) / share;
    const int per = (p.tpg + tiles - 1) / tiles;
    const int wg = blockIdx.x % (p.G * per);
    const int rc = blockIdx.x / (p.G * per);
    g = wg / per;
    part = wg % per;
    chunk = rc % p.nch;
    row = rc / p.nch;
    t0 = chunk * p.CL;
    t1 = min(t0 + p.CL, p.L);
    const int tile = part * tiles + wave;
    const int c = tile * 64 + lane;
    idle = tile >= p.tpg;
    on = c < p.Dg;
    d = g * p.Dg + (on ? c : p.Dg - 1);          // lanes past the group's last channel read it too, and write nothing
  }
};

// NP states of a channel from the n0-th on, of a state tensor [S][D][N] or of A [D][N].  FULL: all of them exist, and a
// lane's come as 16-byte accesses (from and to addresses that need 4-byte alignment only).
template <int NP, bool FULL>
__device__ __forceinline__ void load_state(const float* s, int64_t seq, const ScanArgs& p, int d, float (&h)[NP],
                                           int n0 = 0) {
  const float* q = s + (seq * p.D + d) * p.N + n0;
  if (FULL) {
#pragma unroll
    for (int n = 0; n < NP; n += 4) {
      const Pack<float, 4> v = *reinterpret_cast<const Pack<float, 4>*>(q + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[n + i] = v.v[i];
    }
  } else {
#pragma unroll
    for (int n = 0; n < NP; ++n) h[n] = n0 + n < p.N ? q[n] : 0.f;
  }
}
template <int NP, bool FULL>
__device__ __forceinline__ void store_state(float* s, int64_t seq, const ScanArgs& p, int d, const float (&h)[NP],
                                            int n0 = 0) {
  float* q = s + (seq * p.D + d) * p.N + n0;
  if (FULL) {
#pragma unroll
    for (int n = 0; n < NP; n += 4) {
      const Pack<float, 4> v = {{h[n], h[n + 1], h[n + 2], h[n + 3]}};
      *reinterpret_cast<Pack<float, 4>*>(q + n) = v;
    }
  } else {
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (n0 + n < p.N) q[n] = h[n];
  }
}
template <int NP, bool FULL>
__device__ __forceinline__ void load_rates(const ScanArgs& p, int d, float (&a)[NP], int n0 = 0) {
  load_state<NP, FULL>(p.A, 0, p, d, a, n0);
#pragma unroll
  for (int n = 0; n < NP; ++n) a[n] = decay_rate(a[n]);
}

// the state that a sequence starts with
template <int NP, bool FULL>
__device__ __forceinline__ void entering_state(const ScanArgs& p, int64_t seq, int d, float (&h)[NP], int n0 = 0) {
  if (p.state0) load_state<NP, FULL>(p.state0, seq, p, d, h, n0);
  else {
#pragma unroll
    for (int n = 0; n < NP; ++n) h[n] = 0.f;
  }
}

// An element of a row: wave-uniform address of the row, the lane's place in it in bytes.  The address is kept in scalar
// registers (else the compiler adds the lane's place first, once, and the row's in 64-bit vector arithmetic per access).
#define DVAE_GLOBAL __attribute__((address_space(1)))
template <typename T> __device__ __forceinline__ T lane_load(const T* row, uint32_t at) {
  uint64_t r = (uint64_t)row;
  asm("" : "+s"(r));
  return *(const DVAE_GLOBAL T*)((const DVAE_GLOBAL char*)r + at);
}
template <typename T> __device__ __forceinline__ void lane_store(T* row, uint32_t at, T v) {
  uint64_t r = (uint64_t)row;
  asm("" : "+s"(r));
  *(DVAE_GLOBAL T*)((DVAE_GLOBAL char*)r + at) = v;
}

// The states of a slot, FULL: all NP of them, else the first N.  One scalar address and running offsets, computed anew at
// every call: addresses of their own are kept from block to block, in scalar registers that spill (backward 534 us, with
// this 497), and offsets that are not made anew in vector registers (outputs 162 -> 175 us: a wave less per SIMD).
template <int NP, bool FULL>
__device__ __forceinline__ void load_slot(const float* slot, const ScanArgs& p, int d, float (&h)[NP], int N) {
  uint32_t at = d * 4u;
  asm volatile("" : "+v"(at));
#pragma unroll
  for (int n = 0; n < NP; ++n, at += p.D * 4u) h[n] = FULL || n < N ? lane_load(slot, at) : 0.f;
}
template <int NP, bool FULL>
__device__ __forceinline__ void store_slot(float* slot, const ScanArgs& p, int d, const float (&h)[NP], int N) {
  uint32_t at = d * 4u;
  asm volatile("" : "+v"(at));
#pragma unroll
  for (int n = 0; n < NP; ++n, at += p.D * 4u)
    if (FULL || n < N) lane_store(slot, at, h[n]);
}
__device__ __forceinline__ float* enter_slot(const ScanArgs& p, int row, int chunk) {
  return p.enter + ((int64_t)row * p.enter_row + (int64_t)chunk * p.enter_step) * p.N * p.D;
}
__device__ __forceinline__ float* leave_slot(const ScanArgs& p, int row, int chunk) {
  return p.leave + ((int64_t)row * p.nch + chunk) * p.N * p.D;
}

// One tensor's element of a channel, token by token within a block: the block's row as a scalar address, the lane's place
// in it and the tokens passed as a 32-bit offset, so that eight loads take one scalar address between them (a scalar
// address each, requested together, spilled a hundred scalar registers).
template <typename T> struct Rows {
  const T* base;       // row of the block's first token
  uint32_t step;       // bytes from token to token (the host checked that a block's rows span less than 2 GiB)
  __device__ __forceinline__ Rows(const void* p, int64_t sb, int64_t st, int row, int t0)
      : base((const T*)p + row * sb + t0 * st), step((uint32_t)st * (uint32_t)sizeof(T)) {}
  __device__ __forceinline__ void next() { base = (const T*)((const char*)base + step * SCAN_Q); }
  __device__ __forceinline__ void prev() { base = (const T*)((const char*)base - step * SCAN_Q); }
  // K tokens of the block from the j0-th on; those past the n-th are the n-th again
  template <int K> __device__ __forceinline__ void load(T (&v)[K], int n, uint32_t at, int j0 = 0) const {
    uint64_t r = (uint64_t)base;
    asm("" : "+s"(r));           // (keeps the compiler from adding the lane's place to it)
    at += (uint32_t)max(min(j0, n - 1), 0) * step;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      v[j] = *(const DVAE_GLOBAL T*)((const DVAE_GLOBAL char*)r + at);
      at += j0 + j + 1 < n ? step : 0u;
    }
  }
};

static __device__ const float no_input[SCAN_MAX_N] = {};     // B where there is no token

// STATE_ONLY: the chunk's last state from a zero start, into the next chunk's slot; else the outputs.
//
// A block's inputs were requested a block ahead, B and C are a token ahead.  Lanes past the group's last channel compute
// that channel too and store the same values to the same places, so that no store depends on the lane.  Without packed
// sequences a block is straight-line code: tokens past the chunk's last repeat the last one with a step size of 0 and a B of
// zeros, which leaves the state as it is and stores the same output again.  What packed sequences' borders need stands
// behind wave-uniform branches, and so do their chunks' ends.  (Branches for both: 8 x 2048 x 2048 training 8 % slower.)
//
// Bound by vector arithmetic: a state of a token takes five issue slots in the state pass (two of them the exponential) and
// six in the output pass, a channel's token about 25 more (softplus, gate, conversions).  8 x 2048 x 2048 bf16, N = 16:
// states 110 us, of which 80 are issue slots; outputs 156 us, of which 119, while it reads 201 MB and writes 335, 268 of them
// kept states (3.4 TB/s).  1 x 4096 x 2048: 33 and 42 us.  256 x 20 x 1024 fp32 (one chunk): 42 us.
template <typename T, int NP, bool PACKED, bool FAST, bool STATE_ONLY>
__global__ void __launch_bounds__(256) scan_fwd_kernel(ScanArgs p) {
  const Tile w(p);
  if (w.idle || (STATE_ONLY && w.chunk + 1 == p.nch)) return;
  const int row = w.row;
  const bool gated = p.z != nullptr, plus = p.softplus;
  const uint32_t at = w.d * (uint32_t)sizeof(T);
  Rows<T> ur(p.u, p.u_sb, p.u_st, row, w.t0), dr(p.delta, p.delta_sb, p.delta_st, row, w.t0);
  Rows<T> zr(gated ? p.z : p.u, gated ? p.z_sb : p.u_sb, gated ? p.z_st : p.u_st, row, w.t0);
  T un[SCAN_Q], dn[SCAN_Q], zn[SCAN_Q];            // the block ahead
  BCAhead<T, NP, FAST> ahead;
  ur.load(un, w.t1 - w.t0, at);
  dr.load(dn, w.t1 - w.t0, at);
  if (!STATE_ONLY) zr.load(zn, w.t1 - w.t0, at);
  float A2[NP], h[NP];
  load_rates<NP, FAST>(p, w.d, A2);
#pragma unroll
  for (int n = 0; n < NP; ++n) h[n] = 0.f;
  if (!STATE_ONLY && w.chunk > 0) load_slot<NP, FAST>(enter_slot(p, row, w.chunk), p, w.d, h, p.N);
  if (!PACKED && w.chunk == 0) entering_state<NP, FAST>(p, row, w.d, h);
  const float Dp = p.Dp ? p.Dp[w.d] : 0.f, bias = p.bias ? p.bias[w.d] : 0.f;
  const T* B = (const T*)p.B + row * p.B_sb + w.g * p.B_sg;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  const T *Bt = B + w.t0 * p.B_st, *Ct = C + w.t0 * p.C_st;      // the token ahead
  // A block's first token is requested by the block before it, but not where B and C of two tokens are 64 scalar registers
  // (8 x 2048 x 2048 fp32, outputs: 199 us with it, 184 without; bf16, 1 x 4096: 43 and 45 us).
  constexpr bool CARRY = STATE_ONLY || sizeof(T) * NP < 64;
  constexpr bool FILLS = !PACKED && !STATE_ONLY;   // (the state pass leaves the last chunk out, and the others are whole blocks)
  if (STATE_ONLY) ahead.request_b(Bt, p.N);
  else if (CARRY) ahead.request(Bt, Ct, p.N);
  T* out = (T*)p.out + (int64_t)row * p.L * p.D;
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};
  if (PACKED) q.seek(w.t0);
  float total = 0.f;
  bool cut = false;
  T bc = {};
  for (int t0 = w.t0; t0 < w.t1; t0 += SCAN_Q) {
    const int n = min(SCAN_Q, w.t1 - t0);
    if (!STATE_ONLY) touched(bc);
    T ub[SCAN_Q], pb[SCAN_Q], zb[SCAN_Q];
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) { ub[j] = un[j]; pb[j] = dn[j]; if (!STATE_ONLY) zb[j] = zn[j]; }
    const int left = w.t1 - t0 - SCAN_Q;
    if (left > 0) { ur.next(); dr.next(); zr.next(); }
    ur.load(un, left, at);                         // (the same block again where it was the last)
    dr.load(dn, left, at);
    if (!STATE_ONLY) zr.load(zn, left, at);
    if (!STATE_ONLY && left > 0) {
      const int64_t t = t0 + SCAN_Q;
      bc = touch_rows(B + t * p.B_st, p.B_st, C + t * p.C_st, p.C_st, left, p.N, w.lane);
    }
    if (!STATE_ONLY && p.ckpt)
      store_slot<NP, FAST>(p.ckpt + ((int64_t)row * p.blocks + t0 / SCAN_Q) * p.N * p.D, p, w.d, h, p.N);
    Marks m = {0u, 0u, 0u};
    if (PACKED) m = block_marks(q, t0, n);
    T* ot = out + (int64_t)t0 * p.D;
    uint32_t to = at;
    if (!CARRY) ahead.request(Bt, Ct, p.N);
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) {
      if (PACKED && j >= n) continue;
      const bool there = PACKED || j < n;
      BCAhead<T, NP, FAST> now = ahead;
      float Bv[NP], Cv[NP];
      // behind the chunk's last token: its C again, and a B of zeros, so that B's infinities stay out of the state
      if (FILLS && FAST) Bt = t0 + j + 1 < w.t1 ? Bt + p.B_st : (const T*)no_input;
      else Bt += t0 + j + 1 < w.t1 ? p.B_st : 0;
      Ct += t0 + j + 1 < w.t1 ? p.C_st : 0;
      if (STATE_ONLY) {
        now.arrived_b(Bt);
        ahead.request_b(Bt, p.N);
        now.get_b(Bv);
      } else {
        now.arrived(Bt, Ct);
        if (CARRY || j + 1 < SCAN_Q) ahead.request(Bt, Ct, p.N);
        now.get(Bv, Cv);
      }
      if (FILLS && !FAST) {
#pragma unroll
        for (int i = 0; i < NP; ++i) Bv[i] = there ? Bv[i] : 0.f;
      }
      if (PACKED && !(m.valid >> j & 1)) {
        if (!STATE_ONLY) lane_store(ot, to, from_f32<T>(0.f));
        to += p.D * (uint32_t)sizeof(T);
        continue;
      }
      if (PACKED && (m.start >> j & 1)) {
        entering_state<NP, FAST>(p, q.seq(), w.d, h);
        cut = true;
      }
      const float uu = to_f32(ub[j]);
      const float pre = to_f32(pb[j]) + bias;
      const float sp = softplus_hw(pre);
      const float dt = there ? (plus ? sp : pre) : 0.f;
      const float x = there ? dt * uu : 0.f;       // (0 also where u is infinite)
      float a[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) a[i] = exp2_hw(dt * A2[i]);
      if (STATE_ONLY) {
        __builtin_amdgcn_sched_barrier(0);         // (all of them first: 39 -> 36 us at 1 x 4096 x 2048)
        total += dt;
#pragma unroll
        for (int i = 0; i < NP; ++i) h[i] = fmaf(a[i], h[i], x * Bv[i]);
      } else {
        float y = Dp * uu;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          h[i] = fmaf(a[i], h[i], x * Bv[i]);
          y = fmaf(Cv[i], h[i], y);
        }
        const float zz = to_f32(zb[j]);
        const float gate = zz * sigmoid_hw(zz);
        lane_store(ot, to, from_f32<T>(gated ? y * gate : y));
        to += j + 1 < n ? p.D * (uint32_t)sizeof(T) : 0u;
      }
      if (PACKED && (m.end >> j & 1)) {
        if (!STATE_ONLY && p.state1 && w.on) store_state<NP, FAST>(p.state1, q.seq(), p, w.d, h);
        q.next(t0 + j + 1);
      }
    }
  }
  if (STATE_ONLY) {
    if (w.on) {
      store_slot<NP, FAST>(enter_slot(p, row, w.chunk + 1), p, w.d, h, p.N);
      p.sumdt[((int64_t)row * p.nch + w.chunk) * p.D + w.d] = total;
    }
    if (w.g == 0 && w.part == 0 && threadIdx.x == 0) p.keep[row * p.nch + w.chunk] = cut ? 0.f : 1.f;
  } else if (!PACKED && p.state1 && w.on && w.chunk + 1 == p.nch) {
    store_state<NP, FAST>(p.state1, row, p, w.d, h);
  } else if (PACKED && p.state1) {              // sequences without tokens end with what they entered with
    q.for_empty(w.chunk, p.nch, [&](int s) {
      entering_state<NP, FAST>(p, s, w.d, h);
      if (w.on) store_state<NP, FAST>(p.state1, s, p, w.d, h);
    });
  }
}

// The states (or, BACK, the adjoints) that enter the chunks: x = decay * x + own, along the axis.  Where a sequence
// starts inside a chunk nothing of what enters it gets through.  Bound by the wait for memory, so a workgroup takes 64
// elements and WAVES * JOIN_AHEAD chunks at a time, all requested at once: a wave runs through its JOIN_AHEAD chunks
// from zero, the waves' ends are joined through LDS, and each runs through its chunks again from what really enters them.
// 64 chunks of 2048 channels x 16 states: 7 us; 16 chunks of 8 x 2048 x 16: 13 us (67 MB).
#define JOIN_AHEAD 16
template <bool BACK, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) scan_join_kernel(ScanArgs p) {
  __shared__ float end[WAVES][3][64];         // [wave][own, decay, 1 if nothing gets through][lane]
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t ND = (int64_t)p.N * p.D;
  const int per = (int)((ND + 63) / 64), row = blockIdx.x / per;
  const int64_t i = min((int64_t)(blockIdx.x % per) * 64 + lane, ND - 1);      // (lanes past the last do as it does)
  const int d = (int)(i % p.D), n = (int)(i / p.D);
  const float A2 = decay_rate(p.A[(int64_t)d * p.N + n]);
  const float* sumdt = p.sumdt + (int64_t)row * p.nch * p.D + d;
  float x = 0.f;                                   // what enters the chunks of this round
  for (int k0 = 0; k0 + 1 < p.nch; k0 += WAVES * JOIN_AHEAD) {
    const int kw = k0 + wave * JOIN_AHEAD;
    float own[JOIN_AHEAD], dec[JOIN_AHEAD], keep[JOIN_AHEAD];
    float X = 0.f, P = 1.f, cut = 0.f;
    if (kw + 1 < p.nch) {
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j) {
        const int k = min(kw + j, p.nch - 2);
        const int c = BACK ? p.nch - 1 - k : k;              // the chunk that x passes through
        own[j] = (BACK ? leave_slot(p, row, c - 1) : enter_slot(p, row, c + 1))[i];
        dec[j] = sumdt[(int64_t)c * p.D];
        keep[j] = uniform_load(p.keep, (int64_t)row * p.nch + c);
      }
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j) {
        if (kw + j + 1 < p.nch) {
          const bool through = keep[j] != 0.f;
          dec[j] = exp2_hw(dec[j] * A2);
          X = through ? fmaf(dec[j], X, own[j]) : own[j];
          P = through ? P * dec[j] : 0.f;
          cut = through ? cut : 1.f;
        }
      }
    }
    end[wave][0][lane] = X;
    end[wave][1][lane] = P;
    end[wave][2][lane] = cut;
    __syncthreads();
    float mine = x;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      if (v == wave) mine = x;
      x = end[v][2][lane] != 0.f ? end[v][0][lane] : fmaf(end[v][1][lane], x, end[v][0][lane]);
    }
    __syncthreads();
    if (kw + 1 < p.nch) {
#pragma unroll
      for (int j = 0; j < JOIN_AHEAD; ++j) {
        const int k = kw + j;
        if (k + 1 < p.nch) {
          const int c = BACK ? p.nch - 1 - k : k;
          mine = keep[j] != 0.f ? fmaf(dec[j], mine, own[j]) : own[j];
          (BACK ? leave_slot(p, row, c - 1) : enter_slot(p, row, c + 1))[i] = mine;
        }
      }
    }
  }
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
#define DPP_HALF_MIRROR 0x141
#define DPP_ROR8 0x128
#define DPP_XOR2 0x4e     // quad_perm [2,3,0,1]
#define DPP_XOR1 0xb1     // quad_perm [1,0,3,2]

// Sums of 16 values over the 64 lanes, all at once: a step adds the two halves of the wave (then of a half, ...) and lets
// one half go on with one value, the other with another, so the number of values halves with the number of lanes that
// still hold parts of one.  The sum of value sum_index(lane) ends up in `lane`, in four lanes alike.
__device__ __forceinline__ int sum_index(int lane) { return lane >> 2; }
__device__ __forceinline__ float wave_sums16(float (&v)[16], int lane) {
  // 32 lanes apart, then 16: the swaps exchange the upper half of one register with the lower half of the other
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 8]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float a = lane & 8 ? v[i + 2] : v[i], b = lane & 8 ? v[i] : v[i + 2];
    v[i] = a + dpp<DPP_ROR8>(b);
  }
  const float a = lane & 4 ? v[1] : v[0], b = lane & 4 ? v[0] : v[1];
  float s = a + dpp<DPP_HALF_MIRROR>(b);
  s += dpp<DPP_XOR2>(s);
  return s + dpp<DPP_XOR1>(s);
}

// The adjoint that leaves a chunk to the left if nothing enters it from the right: the sum of C[n] g of its tokens up to
// the first start of a sequence, each through the decays from the chunk's first token to its own: the exponential of the
// step sizes added up so far, so no token waits for another.  8 x 2048 x 2048 bf16: 134 us, 90 of them issue slots.
template <typename T, int NP, bool PACKED, bool FAST>
__global__ void __launch_bounds__(256) scan_bwd_state_kernel(ScanArgs p) {
  const Tile w(p);
  if (w.idle || w.chunk == 0) return;
  const int row = w.row;
  float A2[NP], x[NP];
  load_rates<NP, FAST>(p, w.d, A2);
#pragma unroll
  for (int n = 0; n < NP; ++n) x[n] = 0.f;
  const float bias = p.bias ? p.bias[w.d] : 0.f;
  const bool gated = p.z != nullptr, plus = p.softplus;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  const uint32_t at = w.d * (uint32_t)sizeof(T);
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};
  if (PACKED) q.seek(w.t0);
  float total = 0.f;
  bool cut = false;
  Rows<T> dr(p.delta, p.delta_sb, p.delta_st, row, w.t0), gr(p.dout, p.dout_sb, p.dout_st, row, w.t0);
  Rows<T> zr(gated ? p.z : p.dout, gated ? p.z_sb : p.dout_sb, gated ? p.z_st : p.dout_st, row, w.t0);
  T dn[SCAN_Q], zn[SCAN_Q], gn[SCAN_Q];            // the block ahead
  BCAhead<T, NP, FAST> ahead;
  const T* Ct = C + w.t0 * p.C_st;                 // the token ahead
  ahead.request_b(Ct, p.N);
  dr.load(dn, w.t1 - w.t0, at);
  zr.load(zn, w.t1 - w.t0, at);
  gr.load(gn, w.t1 - w.t0, at);
  for (int t0 = w.t0; t0 < w.t1 && !cut; t0 += SCAN_Q) {
    const int n = min(SCAN_Q, w.t1 - t0);
    T pb[SCAN_Q], zb[SCAN_Q], gb[SCAN_Q];
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) { pb[j] = dn[j]; zb[j] = zn[j]; gb[j] = gn[j]; }
    const int left = w.t1 - t0 - SCAN_Q;
    if (left > 0) { dr.next(); zr.next(); gr.next(); }
    dr.load(dn, left, at);
    zr.load(zn, left, at);
    gr.load(gn, left, at);
    Marks m = {0u, 0u, 0u};
    if (PACKED) m = block_marks(q, t0, n);
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) {
      if (PACKED && (j >= n || cut)) continue;
      const bool there = PACKED || j < n;
      BCAhead<T, NP, FAST> now = ahead;
      float Cv[NP];
      Ct += t0 + j + 1 < w.t1 ? p.C_st : 0;
      now.arrived_b(Ct);
      ahead.request_b(Ct, p.N);
      now.get_b(Cv);
      if (PACKED && !(m.valid >> j & 1)) continue;
      if (PACKED && (m.start >> j & 1)) { cut = true; continue; }
      const float pre = to_f32(pb[j]) + bias;
      const float sp = softplus_hw(pre);
      total += there ? (plus ? sp : pre) : 0.f;
      const float zz = to_f32(zb[j]), gate = zz * sigmoid_hw(zz);
      float g = to_f32(gb[j]);
      g = there ? (gated ? g * gate : g) : 0.f;
#pragma unroll
      for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), Cv[i] * g, x[i]);
      if (PACKED && (m.end >> j & 1)) {
        if (p.dstate1) {
          float e[NP];
          load_state<NP, FAST>(p.dstate1, q.seq(), p, w.d, e);
#pragma unroll
          for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), e[i], x[i]);
        }
        q.next(t0 + j + 1);
      }
    }
  }
  if (!PACKED && p.dstate1 && w.chunk + 1 == p.nch) {
    float e[NP];
    load_state<NP, FAST>(p.dstate1, row, p, w.d, e);
#pragma unroll
    for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), e[i], x[i]);
  }
  if (w.on) {
    store_slot<NP, FAST>(leave_slot(p, row, w.chunk - 1), p, w.d, x, p.N);
    p.sumdt[((int64_t)row * p.nch + w.chunk) * p.D + w.d] = total;
  }
  if (w.g == 0 && w.part == 0 && threadIdx.x == 0) p.keep[row * p.nch + w.chunk] = cut ? 0.f : 1.f;
}

// The states of a tile are shared out over SHARE = NP / 8 waves, eight states each: what one wave keeps of a block (the
// states before its tokens and the decays, computed once for both directions) then fits 256 registers, so that two waves
// run per SIMD and fill each other's waits; with sixteen states in a wave it took 480 and ran alone (8 x 2048 x 2048 bf16:
// 790 against 651 us).  What a channel's token needs besides its states, each wave of a tile does for its share of the
// block's tokens: it loads their inputs, computes their step sizes and gates for the others, and finishes their gradients
// from the waves' parts of y, of the sum of dh B and of that of k A, all by way of LDS.
//
// Bound by vector arithmetic: 177 instructions per token and wave (8 states of 64 channels), 47 slots of them the sums over
// the lanes.  8 x 2048 x 2048 bf16: 496 us, of which 355 are issue slots at two waves per SIMD; it moves 0.77 GB.  256 x 20
// x 1024 fp32: 103 us.  Without keeping the decays three waves would fit a SIMD but for spilled registers: 927 us.  Two
// tiles per workgroup, not four: fewer waves wait at a barrier (four: 6 % slower; one: 2 %, and twice the partial rows).
#define SCAN_NW 8
#define SCAN_BT 2      // tiles per workgroup
template <typename T, int NP, bool PACKED, bool FAST>
__global__ void __launch_bounds__(64 * SCAN_BT * (NP / SCAN_NW), 2) scan_bwd_kernel(ScanArgs p) {
  constexpr int SHARE = NP / SCAN_NW, OWN = SCAN_Q / SHARE;      // waves per tile; tokens of a block that a wave finishes
  __shared__ float red[SCAN_Q][SCAN_BT][2 * NP];                       // [token][tile][dB, dC]
  __shared__ float part[SCAN_Q][3][SCAN_BT * SHARE][64];               // [token][y, dh B, k A][wave][lane]
  __shared__ float in[SCAN_Q][3][SCAN_BT][64];                         // [token][dt, dt u, g][tile][lane]
  const Tile w(p, SCAN_BT, SHARE);
  const int row = w.row, wv = uniform(threadIdx.x >> 6), half = wv % SHARE, n0 = half * SCAN_NW, j0 = half * OWN;
  const bool idle = w.idle;                     // such a wave only takes part in the sums
  const int Nw = min(max(p.N - n0, 0), SCAN_NW);   // states that this wave has
  float A2[SCAN_NW], dh[SCAN_NW], dA[SCAN_NW];
  load_rates<SCAN_NW, FAST>(p, w.d, A2, n0);
#pragma unroll
  for (int i = 0; i < SCAN_NW; ++i) dh[i] = dA[i] = 0.f;
  const int64_t skip = (int64_t)n0 * p.D;          // this wave's rows of a slot
  if (w.chunk + 1 < p.nch) load_slot<SCAN_NW, FAST>(leave_slot(p, row, w.chunk) + skip, p, w.d, dh, Nw);
  else if (!PACKED && p.dstate1) load_state<SCAN_NW, FAST>(p.dstate1, row, p, w.d, dh, n0);
  float dD = 0.f, dbias = 0.f;
  const float Dp = p.Dp ? p.Dp[w.d] : 0.f, bias = p.bias ? p.bias[w.d] : 0.f;
  const bool gated = p.z != nullptr, plus = p.softplus;
  const T* B = (const T*)p.B + row * p.B_sb + w.g * p.B_sg + n0;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg + n0;
  const int64_t flat = (int64_t)row * p.L;
  const uint32_t at = w.d * (uint32_t)sizeof(T);
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};      // the sequence that the way back is in
  if (PACKED) {                                             // the last one that has a token before the chunk's end
    q.seek(w.t1 - 1);
    if (q.s >= q.S || q.b >= w.t1) q.prev(w.t1 - 1);
  }
  const int first = w.t0 + (w.t1 - w.t0 - 1) / SCAN_Q * SCAN_Q;
  const float* ck = p.ckpt + ((int64_t)row * p.blocks + first / SCAN_Q) * p.N * p.D + skip;
  Rows<T> ur(p.u, p.u_sb, p.u_st, row, first), dr(p.delta, p.delta_sb, p.delta_st, row, first);
  Rows<T> gr(p.dout, p.dout_sb, p.dout_st, row, first);
  // (without z, dout is read in its place and not used)
  Rows<T> zr(gated ? p.z : p.dout, gated ? p.z_sb : p.dout_sb, gated ? p.z_st : p.dout_st, row, first);
  T un[OWN], dn[OWN], zn[OWN], gn[OWN], bc = {};      // this wave's tokens of the block ahead,
  float hn[SCAN_NW];                                  // and the state that enters it
  ur.load(un, w.t1 - first, at, j0);
  dr.load(dn, w.t1 - first, at, j0);
  zr.load(zn, w.t1 - first, at, j0);
  gr.load(gn, w.t1 - first, at, j0);
  load_slot<SCAN_NW, FAST>(ck, p, w.d, hn, Nw);

  for (int t0 = first; t0 >= w.t0; t0 -= SCAN_Q) {
    const int n = min(SCAN_Q, w.t1 - t0);
    touched(bc);
    float hs[SCAN_Q + 1][SCAN_NW];
    float dt_[OWN], slope[OWN], u_[OWN], z_[OWN], g_[OWN];      // of this wave's tokens
#pragma unroll
    for (int i = 0; i < SCAN_NW; ++i) hs[0][i] = hn[i];
    BCAhead<T, SCAN_NW, FAST> ahead;
    const T *Bt = B + t0 * p.B_st, *Ct = C + t0 * p.C_st;
    ahead.request_b(Bt, Nw);
    SeqWalk f = q;                                 // the sequence that the states' second computation is in
    Marks m = {0u, 0u, 0u};
    if (PACKED) {
      if (q.s < 0 || q.b > t0 || q.e <= t0) f.seek(t0);
      m = block_marks(f, t0, n);
    }
    // Requests the block before this one.  Called when half of this one's tokens are done, whose registers it takes.
    auto request = [&]() {
      if (t0 > w.t0) {
        ck -= (int64_t)p.N * p.D;
        ur.prev(); dr.prev(); zr.prev(); gr.prev();
      }
      const int left = t0 > w.t0 ? SCAN_Q : n;
      const int64_t t = t0 > w.t0 ? t0 - SCAN_Q : t0;
      bc = touch_rows(B + t * p.B_st, p.B_st, C + t * p.C_st, p.C_st, left, Nw, w.lane);
      ur.load(un, left, at, j0);
      dr.load(dn, left, at, j0);
      zr.load(zn, left, at, j0);
      gr.load(gn, left, at, j0);
      load_slot<SCAN_NW, FAST>(ck, p, w.d, hn, Nw);
    };
#pragma unroll
    for (int jj = 0; jj < OWN; ++jj) {
      // tokens past the chunk's last have a step size and a gradient of 0, which changes nothing, and so have lanes past
      // the group's last channel, which keeps them out of the sums over the channels
      const bool there = j0 + jj < n && w.on;
      const float pre = to_f32(dn[jj]) + bias;
      const float sp = softplus_hw(pre, slope[jj]);
      dt_[jj] = there ? (plus ? sp : pre) : 0.f;
      slope[jj] = plus ? slope[jj] : 1.f;
      u_[jj] = to_f32(un[jj]);
      z_[jj] = to_f32(zn[jj]);
      g_[jj] = there ? to_f32(gn[jj]) : 0.f;
      in[j0 + jj][0][w.wave][w.lane] = dt_[jj];
      in[j0 + jj][1][w.wave][w.lane] = there ? dt_[jj] * u_[jj] : 0.f;      // (0 also where u is infinite)
      in[j0 + jj][2][w.wave][w.lane] = gated ? g_[jj] * (z_[jj] * sigmoid_hw(z_[jj])) : g_[jj];
    }
    __syncthreads();                               // and everyone has read the sums of the block behind
    float a[SCAN_Q][SCAN_NW];
    // What is read from LDS is read a token ahead too, beside the request for B and C: waiting for LDS alone is not
    // possible while scalar loads are on the way.
    float dtn = in[0][0][w.wave][w.lane], xn = in[0][1][w.wave][w.lane], gn_ = 0.f;
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) {
#pragma unroll
      for (int i = 0; i < SCAN_NW; ++i) hs[j + 1][i] = hs[j][i];
      if (PACKED && j >= n) continue;
      BCAhead<T, SCAN_NW, FAST> now = ahead;
      float Bv[SCAN_NW];
      const bool more = j + 1 < SCAN_Q && (!PACKED || j + 1 < n);
      Bt += j + 1 < n ? p.B_st : 0;
      Ct += j + 1 < n ? p.C_st : 0;
      now.arrived_b(Bt);
      if (more) ahead.request_b(Bt, Nw);
      else ahead.request(Bt, Ct, Nw);              // the last token's, where the way back begins
      now.get_b(Bv);
      const float dt = dtn, x = xn;
      const int next = more ? j + 1 : j;
      dtn = in[next][0][w.wave][w.lane];
      xn = in[next][1][w.wave][w.lane];
      gn_ = in[next][2][w.wave][w.lane];
      if (PACKED && !(m.valid >> j & 1)) continue;
      if (PACKED && (m.start >> j & 1)) entering_state<SCAN_NW, FAST>(p, f.seq(), w.d, hs[j + 1], n0);
#pragma unroll
      for (int i = 0; i < SCAN_NW; ++i) {
        a[j][i] = exp2_hw(dt * A2[i]);
        hs[j + 1][i] = fmaf(a[j][i], hs[j + 1][i], x * Bv[i]);
      }
      if (PACKED && (m.end >> j & 1)) f.next(t0 + j + 1);
      __builtin_amdgcn_sched_barrier(0);           // (mixing tokens spills registers: 808 against 580 us)
    }
#pragma unroll
    for (int j = SCAN_Q - 1; j >= 0; --j) {
      if (j == SCAN_Q / 2 - 1) request();
      if (PACKED && j >= n) continue;
      if (!PACKED && j + 1 < SCAN_Q && j + 1 == n) {
        // What the tokens that fill the row's last block up have added: 0, or NaN where the last state is infinite.  (The
        // block is the first one here.  8 x 2048 x 2048 bf16 training 826 us without this, 837 with it; 893 if a branch leaves
        // those tokens out; 868 to 872 if an infinite C is kept out of the adjoint as well.)
#pragma unroll
        for (int i = 0; i < SCAN_NW; ++i) dA[i] = 0.f;
      }
      BCAhead<T, SCAN_NW, FAST> now = ahead;
      float Bv[SCAN_NW], Cv[SCAN_NW];
      Bt -= j > 0 && j < n ? p.B_st : 0;
      Ct -= j > 0 && j < n ? p.C_st : 0;
      now.arrived(Bt, Ct);
      if (j > 0) ahead.request(Bt, Ct, Nw);
      now.get(Bv, Cv);
      const float dt = dtn, x = xn, g = gn_;
      if (j > 0) {
        dtn = in[j - 1][0][w.wave][w.lane];
        xn = in[j - 1][1][w.wave][w.lane];
        gn_ = in[j - 1][2][w.wave][w.lane];
      }
      const int c = sum_index(w.lane), cell = c < SCAN_NW ? n0 + c : NP + n0 + c - SCAN_NW;      // (four lanes alike)
      if (PACKED && !(m.valid >> j & 1)) {
        red[j][w.wave][cell] = 0.f;
        continue;
      }
      if (PACKED && (m.end >> j & 1)) {
        if (p.dstate1) load_state<SCAN_NW, FAST>(p.dstate1, q.seq(), p, w.d, dh, n0);
        else {
#pragma unroll
          for (int i = 0; i < SCAN_NW; ++i) dh[i] = 0.f;
        }
      }
      float hb[SCAN_NW];                           // the state before the token
#pragma unroll
      for (int i = 0; i < SCAN_NW; ++i) hb[i] = hs[j][i];
      if (PACKED && (m.start >> j & 1)) entering_state<SCAN_NW, FAST>(p, q.seq(), w.d, hb, n0);
      float y = 0.f, through = 0.f, ka = 0.f, pv[2 * SCAN_NW];
#pragma unroll
      for (int i = 0; i < SCAN_NW; ++i) {
        y = fmaf(Cv[i], hs[j + 1][i], y);
        const float d = fmaf(Cv[i], g, dh[i]);
        pv[i] = d * x;
        pv[SCAN_NW + i] = g * hs[j + 1][i];
        through = fmaf(d, Bv[i], through);
        dh[i] = d * a[j][i];
        const float k = dh[i] * hb[i];
        dA[i] = fmaf(k, dt, dA[i]);
        ka = fmaf(k, A2[i], ka);
      }
      part[j][0][wv][w.lane] = y;
      part[j][1][wv][w.lane] = through;
      part[j][2][wv][w.lane] = ka;
      red[j][w.wave][cell] = wave_sums16(pv, w.lane);
      if (PACKED && (m.start >> j & 1)) {
        if (p.dstate0 && w.on && !idle) store_state<SCAN_NW, FAST>(p.dstate0, q.seq(), p, w.d, dh, n0);
        q.prev(t0 + j - 1);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    const int64_t o = (flat + t0 + j0) * p.D;
    uint32_t to = at;
    asm volatile("" : "+v"(to));
#pragma unroll
    for (int jj = 0; jj < OWN; ++jj) {
      const int j = j0 + jj;
      if (j < n) {
        float du = 0.f, dd = 0.f, dz = 0.f;
        if (!PACKED || (m.valid >> j & 1)) {
          float y = Dp * u_[jj], through = 0.f, ka = 0.f;
#pragma unroll
          for (int k = 0; k < SHARE; ++k) {
            y += part[j][0][w.wave * SHARE + k][w.lane];
            through += part[j][1][w.wave * SHARE + k][w.lane];
            ka += part[j][2][w.wave * SHARE + k][w.lane];
          }
          const float sg = sigmoid_hw(z_[jj]);
          const float g = gated ? g_[jj] * (z_[jj] * sg) : g_[jj];
          dz = g_[jj] * y * sg * fmaf(z_[jj], 1.f - sg, 1.f);
          du = fmaf(through, dt_[jj], Dp * g);
          dd = fmaf(ka, LN2_F, through * u_[jj]) * slope[jj];
          dD = fmaf(g, u_[jj], dD);
          dbias += dd;
        }
        if (w.on && !idle) {
          if (gated) lane_store((T*)p.dz + o, to, from_f32<T>(dz));
          lane_store((T*)p.du + o, to, from_f32<T>(du));
          lane_store((T*)p.ddelta + o, to, from_f32<T>(dd));
        }
      }
      to += (uint32_t)p.D * (uint32_t)sizeof(T);
    }
    const int N = FAST ? NP : p.N;
    for (int i = threadIdx.x; i < n * 2 * N; i += 64 * SCAN_BT * SHARE) {
      const int j = i / (2 * N), c = i % (2 * N), k = c < N ? c : c - N + NP;
      float s = red[j][0][k];
#pragma unroll
      for (int t = 1; t < SCAN_BT; ++t) s += red[j][t][k];
      p.part_bc[(((int64_t)w.part * p.rows * p.L + flat + t0 + j) * p.G + w.g) * 2 * N + c] = s;
    }
  }
  if (!PACKED && w.chunk == 0 && p.dstate0 && w.on && !idle) store_state<SCAN_NW, FAST>(p.dstate0, row, p, w.d, dh, n0);
  __syncthreads();
  part[0][0][wv][w.lane] = dD;
  part[0][1][wv][w.lane] = dbias;
  __syncthreads();
  if (w.on && !idle) {
    float* pa = p.part_a + ((int64_t)row * p.nch + w.chunk) * (p.N + 2) * p.D + w.d;
#pragma unroll
    for (int i = 0; i < SCAN_NW; ++i)
      if (i < Nw) pa[(int64_t)(n0 + i) * p.D] = dA[i];
    if (half == 0) {
#pragma unroll
      for (int k = 1; k < SHARE; ++k) {
        dD += part[0][0][w.wave * SHARE + k][w.lane];
        dbias += part[0][1][w.wave * SHARE + k][w.lane];
      }
      pa[(int64_t)p.N * p.D] = dD;
      pa[(int64_t)(p.N + 1) * p.D] = dbias;
    }
  }
}

// The gradients that are sums of partial rows, in one launch.  The first `bc_groups` workgroups add up dB and dC of every
// token over the backward kernel's workgroups; the others dA [D][N], dD [D] and dbias [D] over rows and chunks.  Always in
// the same order, so results repeat bit for bit.  8 x 2048 x 2048: 14 us for 53 MB.
template <typename T>
__global__ void __launch_bounds__(64 * SUM_WAVES) scan_sums_kernel(ScanArgs p, T* dB, T* dC, float* dA, float* dD,
                                                                   float* dbias, int64_t tokens_g, int parts,
                                                                   unsigned bc_groups) {
  if (blockIdx.x < bc_groups) {
    const int64_t i = (int64_t)blockIdx.x * (64 * SUM_WAVES) + threadIdx.x;
    const int64_t total = tokens_g * 2 * p.N;
    if (i >= total) return;
    float s = 0.f;
    for (int k = 0; k < parts; ++k) s += p.part_bc[k * total + i];
    const int64_t r = i / (2 * p.N);
    const int c = (int)(i % (2 * p.N));
    if (c < p.N) dB[r * p.N + c] = from_f32<T>(s);
    else dC[r * p.N + c - p.N] = from_f32<T>(s);
    return;
  }
  const int64_t total = (int64_t)(p.N + 2) * p.D;
  const int64_t i = (int64_t)(blockIdx.x - bc_groups) * 64 + (threadIdx.x & 63);
  const float s = column_sum(p.part_a, (int64_t)p.rows * p.nch, total, i, i < total);
  if (threadIdx.x >= 64 || i >= total) return;
  const int n = (int)(i / p.D), d = (int)(i % p.D);
  if (n < p.N) { if (dA) dA[(int64_t)d * p.N + n] = s; }
  else if (n == p.N) { if (dD) dD[d] = s; }
  else if (dbias) dbias[d] = s;
}

// One token per row.  Nearly all of the traffic is the state, read and written once: a lane owns four states of a channel
// (one 16-byte access each way where N is a multiple of 4 and all is aligned), a channel's LPC lanes are neighbours, and the
// sum over them takes two lane exchanges.  What a channel reads besides (inputs, step size) its lanes read and compute
// alike.  A lane goes through R rows whose loads are in flight together and share its A.  256 x 2048 x 16 bf16: 19 us for
// 72 MB (3.8 TB/s); 1 x 512: 4 us.
template <typename T, int LPC, int R, bool VEC>
__global__ void __launch_bounds__(256) scan_step_kernel(ScanArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int q = (int)(i % LPC), d = (int)(i / LPC % p.D), n0 = q * 4;
  const int row0 = (int)(i / LPC / p.D) * R;
  if (row0 >= p.rows) return;
  const int g = d / p.Dg;
  float A2[4], h[R][4], Bv[R][4], Cv[R][4], uu[R], pre[R], zz[R];
  const float* A = p.A + (int64_t)d * p.N + n0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(row0 + r, p.rows - 1);            // a row past the last is the last again, and not written
    const float* s = p.state1 + ((int64_t)row * p.D + d) * p.N + n0;
    const T* B = (const T*)p.B + row * p.B_sb + g * p.B_sg + n0;
    const T* C = (const T*)p.C + row * p.C_sb + g * p.C_sg + n0;
    if (VEC && n0 < p.N) {
      load_pack<float, 4>(s, h[r]);
      load_pack<T, 4>(B, Bv[r]);
      load_pack<T, 4>(C, Cv[r]);
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const bool there = n0 + n < p.N;
        h[r][n] = there ? s[n] : 0.f;
        Bv[r][n] = there ? to_f32(B[n]) : 0.f;
        Cv[r][n] = there ? to_f32(C[n]) : 0.f;
      }
    }
    uu[r] = to_f32(((const T*)p.u)[row * p.u_sb + d]);
    pre[r] = to_f32(((const T*)p.delta)[row * p.delta_sb + d]);
    zz[r] = p.z ? to_f32(((const T*)p.z)[row * p.z_sb + d]) : 0.f;
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) A2[n] = n0 + n < p.N ? decay_rate(A[n]) : 0.f;
  const float bias = p.bias ? p.bias[d] : 0.f, Dp = p.Dp ? p.Dp[d] : 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + r;
    const float v = pre[r] + bias, dt = p.softplus ? softplus_hw(v) : v, x = dt * uu[r];
    float y = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      h[r][n] = fmaf(exp2_hw(dt * A2[n]), h[r][n], x * Bv[r][n]);
      y = fmaf(Cv[r][n], h[r][n], y);
    }
    if (LPC >= 2) y += dpp<DPP_XOR1>(y);
    if (LPC >= 4) y += dpp<DPP_XOR2>(y);
    y = fmaf(Dp, uu[r], y);
    if (p.z) y *= zz[r] * sigmoid_hw(zz[r]);
    if (row >= p.rows) continue;
    float* s = p.state1 + ((int64_t)row * p.D + d) * p.N + n0;
    if (VEC) {
      if (n0 < p.N) store_pack<float, 4>(s, h[r]);
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n0 + n < p.N) s[n] = h[r][n];
    }
    if (q == 0) ((T*)p.out)[(int64_t)row * p.D + d] = from_f32<T>(y);
  }
}

// ------------------------------------------------------------------------------------------------ host side
static int scan_check(const char* what, int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N, int64_t S,
                      const int32_t* offsets, int dtype) {
  DVAE_REQUIRE(dtype == DVAE_DT_F32 || dtype == DVAE_DT_BF16, "%s: dtype must be fp32 (0) or bf16 (1)", what);
  DVAE_REQUIRE(rows >= 0 && L >= 0 && D > 0 && G > 0 && D % G == 0, "%s: D must be a multiple of G", what);
  DVAE_REQUIRE(N > 0 && N <= SCAN_MAX_N, "%s: 1 to %d states per channel, got %ld", what, SCAN_MAX_N, (long)N);
  DVAE_REQUIRE(rows < (1ll << 31) && L < (1ll << 31) && rows * L < SEQ_MAX_TOKENS && D < (1ll << 24), "%s: too large",
               what);
  DVAE_REQUIRE(!offsets || (rows == 1 && S >= 1 && S < (1ll << 30)), "%s: offsets go with one row and S >= 1", what);
  return 0;
}

// the kernels step through a block's rows by 32-bit byte offsets
static bool scan_stride_ok(int64_t st) { return st >= 0 && st < (1ll << 31) / (SCAN_Q * 4); }

// rows of partial sums of dB and dC: one per workgroup of the backward kernel within a group
static int scan_bc_parts(int tpg) { return (tpg + SCAN_BT - 1) / SCAN_BT; }

static void scan_shape(ScanArgs& p, int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N, int64_t S) {
  p.rows = (int)rows; p.L = (int)L; p.D = (int)D; p.G = (int)G; p.N = (int)N; p.S = (int)S;
  p.Dg = (int)(D / G);
  p.tpg = (p.Dg + 63) / 64;
  p.wpg = p.G * ((p.tpg + 3) / 4);
  p.blocks = (int)ceil_div64(L, SCAN_Q);
  // Chunks: none where the rows give every SIMD two waves without them, since the passes that chunks need cost more than a
  // third and a fourth wave gain (split against whole, bf16, outputs of 256 x 512 x 2048: 1695 and 872 us).  With 16 states
  // and several rows that is so from three waves for every four SIMDs on (outputs of 24 x 512 x 2048 197 and 201 us, 32 x
  // 1024 x 2048 452 and 395, training of 28 x 4096 x 2048 fp32 6001 and 5136; but 16 x 1024 x 2048, two waves for four SIMDs:
  // outputs 236 and 392).  Fewer states have one wave per tile on the way back, and packed sequences' borders are waits that
  // other waves fill: training of 28 x 2048 x 2048 with 8 states 2143 and 2854 us, of 40 sequences packed into 8192 x 49152
  // fp32 11310 and 14928.
  // Else as many as it takes to reach two waves per SIMD, none shorter than 32 tokens; from there on to four per SIMD, none
  // shorter than 64.  Two against four: 8 x 2048 x 2048 training 914 and 834 us, outputs of 1 x 8192 x 2048 139 and 127 us;
  // 1 x 131072 x 64, where four are 32 tokens each: 160 and 218 us.
  const int64_t waves = rows * p.tpg * G, enough = N == 16 && rows > 1 ? SCAN_WAVES / 8 * 3 : SCAN_WAVES;
  const int64_t two = waves > 0 ? ceil_div64(SCAN_WAVES, waves) : 1, four = 2 * two;
  const int64_t n2 = two < L / 32 ? two : L / 32, n4 = four < L / 64 ? four : L / 64;
  const int64_t n = waves >= enough ? 1 : n2 > n4 ? n2 : n4;
  p.CL = (int)(n > 1 ? ceil_div64(ceil_div64(L, n), SCAN_Q) * SCAN_Q : p.blocks * SCAN_Q);
  p.nch = (int)(L > 0 ? ceil_div64(L, p.CL) : 1);
}

// where the states that enter the chunks lie: among those that training keeps, else in scratch of their own
static float* scan_scratch(ScanArgs& p, float* ws) {
  if (p.ckpt) { p.enter = p.ckpt; p.enter_row = p.blocks; p.enter_step = p.CL / SCAN_Q; }
  else { p.enter = ws; p.enter_row = p.nch; p.enter_step = 1; ws += (int64_t)p.rows * p.nch * p.N * p.D; }
  p.sumdt = ws; ws += (int64_t)p.rows * p.nch * p.D;
  p.keep = ws;
  return ws + (((int64_t)p.rows * p.nch + 3) & ~3ll);
}

// whether every launch is one that the device takes
static bool scan_fits(const ScanArgs& p) {
  const int64_t chunks = (int64_t)p.rows * p.nch;
  return launch_fits(chunks * p.wpg, 256) && launch_fits(chunks * p.G * scan_bc_parts(p.tpg), 256) &&
         (p.nch == 1 || launch_fits(ceil_div64((int64_t)p.N * p.D, 64) * p.rows, p.nch > 2 * JOIN_AHEAD + 1 ? 512 : 64));
}

// whether B and C of every token and group can be read as whole aligned words
static bool scan_words(const ScanArgs& p, int dtype, int NP) {
  if (p.N != NP) return false;
  if (dtype == DVAE_DT_F32) return true;
  const int64_t odd = p.B_sb | p.B_st | p.B_sg | p.C_sb | p.C_st | p.C_sg;
  return !(odd & 1) && !(((uintptr_t)p.B | (uintptr_t)p.C) & 3);
}

// eight waves per workgroup where one would go round more than twice: 126 chunks of 1002 channels 18 -> 9 us, but 16
// chunks of 8 x 2048 channels 10 -> 27 us
template <bool BACK> static void scan_join(const ScanArgs& p, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div64((int64_t)p.N * p.D, 64) * p.rows));
  if (p.nch > 2 * JOIN_AHEAD + 1) DVAE_LAUNCH((scan_join_kernel<BACK, 8>), grid, dim3(64 * 8), 0, s, p);
  else DVAE_LAUNCH((scan_join_kernel<BACK, 1>), grid, dim3(64), 0, s, p);
}
template <typename T, int NP, bool PACKED, bool FAST> static void scan_fwd_launch(const ScanArgs& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.rows * p.nch * p.wpg)), block(256);
  if (p.nch > 1) {
    DVAE_LAUNCH((scan_fwd_kernel<T, NP, PACKED, FAST, true>), grid, block, 0, s, p);
    scan_join<false>(p, s);
  }
  DVAE_LAUNCH((scan_fwd_kernel<T, NP, PACKED, FAST, false>), grid, block, 0, s, p);
}
template <typename T, int NP, bool PACKED, bool FAST> static void scan_bwd_launch(const ScanArgs& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.rows * p.nch * p.wpg)), block(256);
  if (p.nch > 1) {
    DVAE_LAUNCH((scan_bwd_state_kernel<T, NP, PACKED, FAST>), grid, block, 0, s, p);
    scan_join<true>(p, s);
  }
  const int64_t groups = (int64_t)p.rows * p.nch * p.G * scan_bc_parts(p.tpg);
  DVAE_LAUNCH((scan_bwd_kernel<T, NP, PACKED, FAST>), dim3((unsigned)groups), dim3(64 * SCAN_BT * (NP / SCAN_NW)), 0, s, p);
}

#define SCAN_LAUNCH(K, T, NP, p, s)                                                                   \
  do {                                                                                                \
    const bool fast__ = scan_words(p, sizeof(T) == 4 ? DVAE_DT_F32 : DVAE_DT_BF16, NP);               \
    if (p.offsets) {                                                                                  \
      if (fast__) K<T, NP, true, true>(p, s); else K<T, NP, true, false>(p, s);                       \
    } else {                                                                                          \
      if (fast__) K<T, NP, false, true>(p, s); else K<T, NP, false, false>(p, s);                     \
    }                                                                                                 \
  } while (0)
#define SCAN_DISPATCH(K, dtype, p, s)                                                                 \
  do {                                                                                                \
    if (dtype == DVAE_DT_F32) {                                                                       \
      if (p.N <= 8) SCAN_LAUNCH(K, float, 8, p, s); else SCAN_LAUNCH(K, float, 16, p, s);             \
    } else {                                                                                          \
      if (p.N <= 8) SCAN_LAUNCH(K, bf16_t, 8, p, s); else SCAN_LAUNCH(K, bf16_t, 16, p, s);           \
    }                                                                                                 \
  } while (0)

extern "C" int64_t dvae_selective_scan_ckpt_floats(int64_t rows, int64_t L, int64_t D, int64_t N) {
  return rows * ceil_div64(L, SCAN_Q) * N * D;
}

extern "C" int64_t dvae_selective_scan_fwd_ws_floats(int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N, int keep) {
  ScanArgs p = {};
  if (rows * L <= 0 || D <= 0 || G <= 0) return 0;
  scan_shape(p, rows, L, D, G, N, 1);
  return p.nch == 1 ? 0 : rows * p.nch * ((keep ? 1 : N + 1) * D + 1) + 4;
}

extern "C" int64_t dvae_selective_scan_bwd_ws_floats(int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N) {
  ScanArgs p = {};
  if (rows * L <= 0 || D <= 0 || G <= 0) return 0;
  scan_shape(p, rows, L, D, G, N, 1);
  const int64_t parts = scan_bc_parts(p.tpg), chunks = rows * p.nch;
  return parts * rows * L * G * 2 * N + chunks * (N + 2) * D + (p.nch == 1 ? 0 : chunks * ((N + 1) * D + 1) + 4);
}

extern "C" int dvae_selective_scan_fwd(const void* u, int64_t u_sb, int64_t u_st, const void* delta, int64_t delta_sb,
                                       int64_t delta_st, const float* A, const void* B, int64_t B_sb, int64_t B_st,
                                       int64_t B_sg, const void* C, int64_t C_sb, int64_t C_st, int64_t C_sg,
                                       const float* Dp, const void* z, int64_t z_sb, int64_t z_st, const float* bias,
                                       int softplus, const float* state0, float* state1, const int32_t* offsets,
                                       void* out, float* ckpt, int64_t rows, int64_t L, int64_t D, int64_t G, int64_t N,
                                       int64_t S, int dtype, float* ws, dvae_stream_t stream) {
  const int rc = scan_check("selective_scan_fwd", rows, L, D, G, N, S, offsets, dtype);
  if (rc) return rc;
  if (rows * L == 0) return 0;
  if (L == 1) u_st = delta_st = z_st = 0;          // (no token to step to)
  DVAE_REQUIRE(scan_stride_ok(u_st) && scan_stride_ok(delta_st) && scan_stride_ok(z_st),
               "selective_scan_fwd: token strides must be below 2^26 elements");
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.u_st = u_st; p.delta = delta; p.delta_sb = delta_sb; p.delta_st = delta_st; p.A = A;
  p.B = B; p.B_sb = B_sb; p.B_st = B_st; p.B_sg = B_sg; p.C = C; p.C_sb = C_sb; p.C_st = C_st; p.C_sg = C_sg;
  p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.z_st = z_st; p.bias = bias; p.softplus = softplus;
  p.state0 = state0; p.state1 = state1; p.offsets = offsets; p.out = out; p.ckpt = ckpt;
  scan_shape(p, rows, L, D, G, N, S);
  scan_scratch(p, ws);
  DVAE_REQUIRE(scan_fits(p), "selective_scan_fwd: too many rows for one launch");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(rows * L * (double)e * ((z ? 4 : 3) * D + 2 * G * N), DVAE_UNIT_BYTE);
  SCAN_DISPATCH(scan_fwd_launch, dtype, p, ST(stream));
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
  if (L == 1) u_st = delta_st = z_st = dout_st = 0;
  DVAE_REQUIRE(!z || dz, "selective_scan_bwd: dz is needed with z");
  DVAE_REQUIRE(scan_stride_ok(u_st) && scan_stride_ok(delta_st) && scan_stride_ok(z_st) && scan_stride_ok(dout_st),
               "selective_scan_bwd: token strides must be below 2^26 elements");
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.u_st = u_st; p.delta = delta; p.delta_sb = delta_sb; p.delta_st = delta_st; p.A = A;
  p.B = B; p.B_sb = B_sb; p.B_st = B_st; p.B_sg = B_sg; p.C = C; p.C_sb = C_sb; p.C_st = C_st; p.C_sg = C_sg;
  p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.z_st = z_st; p.bias = bias; p.softplus = softplus;
  p.state0 = state0; p.offsets = offsets; p.dout = dout; p.dout_sb = dout_sb; p.dout_st = dout_st;
  p.dstate1 = dstate1; p.dstate0 = dstate0; p.ckpt = const_cast<float*>(ckpt);
  p.du = du; p.ddelta = ddelta; p.dz = dz;
  scan_shape(p, rows, L, D, G, N, S);
  const int parts = scan_bc_parts(p.tpg);
  float* after = scan_scratch(p, ws);
  if (p.nch == 1) after = ws;
  else { p.leave = after; after += (int64_t)rows * p.nch * N * D; }
  p.part_bc = after;
  p.part_a = after + (int64_t)parts * rows * L * G * 2 * N;
  const int64_t bc = rows * L * G, bc_groups = ceil_div64(bc * 2 * N, 64 * SUM_WAVES);
  const int64_t sums = bc_groups + ceil_div64((N + 2) * D, 64);
  DVAE_REQUIRE(scan_fits(p), "selective_scan_bwd: too many rows for one launch");
  DVAE_REQUIRE(launch_fits(sums, 64 * SUM_WAVES), "selective_scan_bwd: too many tokens and groups for one launch");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(rows * L * (double)e * ((z ? 7 : 5) * D + 4 * G * N), DVAE_UNIT_BYTE);
  SCAN_DISPATCH(scan_bwd_launch, dtype, p, ST(stream));
  DVAE_LAUNCH_CHECK("selective_scan_bwd");
#define SCAN_SUMS(T)                                                                                                  \
  DVAE_LAUNCH((scan_sums_kernel<T>), dim3((unsigned)sums), dim3(64 * SUM_WAVES), 0, ST(stream), p, (T*)dB, (T*)dC, dA, \
              dD, dbias, bc, parts, (unsigned)bc_groups)
  if (dtype == DVAE_DT_F32) SCAN_SUMS(float); else SCAN_SUMS(bf16_t);
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
  // four rows per lane where that leaves two workgroups per compute unit: 256 x 2048 x 16, 19 against 22 us
  const int lpc = N > 8 ? 4 : N > 4 ? 2 : 1;
  const bool many = ceil_div64(rows, 4) * D * lpc >= 512 * 256;
  const uintptr_t bc = (uintptr_t)B | (uintptr_t)C;
  const bool vec = N % 4 == 0 && !((uintptr_t)state & 15) && !((B_sb | B_sg | C_sb | C_sg) & 3) &&
                   !(bc & (dtype == DVAE_DT_F32 ? 15 : 7));
  const int64_t grid = ceil_div64(ceil_div64(rows, many ? 4 : 1) * D * lpc, 256);
  DVAE_REQUIRE(launch_fits(grid, 256), "selective_scan_step: too many rows for one launch");
  DVAE_WORK(rows * (double)D * N * 8, DVAE_UNIT_BYTE);
#define SCAN_STEP(T, LPC, R)                                                                               \
  do {                                                                                                     \
    if (vec) DVAE_LAUNCH((scan_step_kernel<T, LPC, R, true>), dim3((unsigned)grid), dim3(256), 0, ST(stream), p); \
    else DVAE_LAUNCH((scan_step_kernel<T, LPC, R, false>), dim3((unsigned)grid), dim3(256), 0, ST(stream), p);    \
  } while (0)
#define SCAN_STEP_N(T, R)                                                                                  \
  do {                                                                                                     \
    if (lpc == 4) SCAN_STEP(T, 4, R); else if (lpc == 2) SCAN_STEP(T, 2, R); else SCAN_STEP(T, 1, R);      \
  } while (0)
  if (dtype == DVAE_DT_F32) { if (many) SCAN_STEP_N(float, 4); else SCAN_STEP_N(float, 1); }
  else { if (many) SCAN_STEP_N(bf16_t, 4); else SCAN_STEP_N(bf16_t, 1); }
  DVAE_LAUNCH_CHECK("selective_scan_step");
  return 0;
}
