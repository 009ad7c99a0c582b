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
#define SCAN_WAVES 2048    // waves that a launch aims at: two per SIMD
#define SCAN_MIN_CHUNK 32  // tokens: below this a chunk's fixed costs (its state in and out) weigh as much as its tokens

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
  int rows, L, D, G, N, S, Dg, tpg, ntiles, wpg, softplus, blocks;
  int nch, CL, enter_row, enter_step;   // chunks, their tokens; slots of `enter` per row and from chunk to chunk
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

// The same, requested ahead.  Scalar loads return in any order, so waiting for one means waiting for all: `arrived`
// makes the words of this token a dependence of the address of the next one's, which puts the wait before the next
// request and a token's arithmetic between a request and its wait.
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
    BCLoad<T, NP, false>::get(B, 0, N, b);
    BCLoad<T, NP, false>::get(C, 0, N, c);
  }
  __device__ __forceinline__ void request_b(const T* B, int N) { BCLoad<T, NP, false>::get(B, 0, N, b); }
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

// One wave: 64 channels of one group, one chunk of one row.  A workgroup's four waves are neighbours in a group.
struct Tile {
  int g, d, lane, wave, part, chunk, row, t0, t1;
  bool on;
  __device__ __forceinline__ explicit Tile(const ScanArgs& p) {
    lane = threadIdx.x & 63;
    wave = uniform(threadIdx.x >> 6);
    const int wg = blockIdx.x % p.wpg;
    const int rc = blockIdx.x / p.wpg;
    const int per = (p.tpg + 3) / 4;
    g = wg / per;
    part = wg % per;
    chunk = rc % p.nch;
    row = rc / p.nch;
    t0 = chunk * p.CL;
    t1 = min(t0 + p.CL, p.L);
    const int c = (part * 4 + wave) * 64 + lane;
    on = c < p.Dg;
    d = g * p.Dg + (on ? c : p.Dg - 1);          // lanes past the group's last channel read it too, and write nothing
  }
  __device__ __forceinline__ bool idle(const ScanArgs& p) const { return part * 4 + wave >= p.tpg; }
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

// FULL: all NP states exist
template <int NP, bool FULL>
__device__ __forceinline__ void load_slot(const float* slot, const ScanArgs& p, int d, float (&h)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; ++n) h[n] = FULL || n < p.N ? lane_load(slot + (int64_t)n * p.D, d * 4u) : 0.f;
}
template <int NP, bool FULL>
__device__ __forceinline__ void store_slot(float* slot, const ScanArgs& p, int d, const float (&h)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; ++n)
    if (FULL || n < p.N) lane_store(slot + (int64_t)n * p.D, d * 4u, h[n]);
}
__device__ __forceinline__ float* enter_slot(const ScanArgs& p, int row, int chunk) {
  return p.enter + ((int64_t)row * p.enter_row + (int64_t)chunk * p.enter_step) * p.N * p.D;
}
__device__ __forceinline__ float* leave_slot(const ScanArgs& p, int row, int chunk) {
  return p.leave + ((int64_t)row * p.nch + chunk) * p.N * p.D;
}

// What a block of tokens reads per channel, as stored.  Tokens past the chunk's last are the last one again.
template <typename T> struct FwdRaw {
  T u[SCAN_Q], dl[SCAN_Q], z[SCAN_Q];
  // from the rows that the pointers are at; they end up at the block's last row
  template <bool Z>
  __device__ __forceinline__ void load(const T*& up, int64_t u_st, const T*& dp, int64_t d_st, const T*& zp, int64_t z_st,
                                       int n, uint32_t at) {
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) {
      u[j] = lane_load(up, at);
      dl[j] = lane_load(dp, at);
      if (Z) z[j] = lane_load(zp, at);
      const bool more = j + 1 < SCAN_Q && j + 1 < n;
      up += more ? u_st : 0;
      dp += more ? d_st : 0;
      if (Z) zp += more ? z_st : 0;
    }
  }
};

// STATE_ONLY: the chunk's last state from a zero start, into the next chunk's slot; else the outputs.
//
// A block of SCAN_Q tokens in which no sequence starts or ends is straight-line code: its inputs were requested a block
// ahead, and the compiler can request B and C tokens ahead.  Nothing in it is conditional.  Lanes past the group's last
// channel compute that channel too and store the same values to the same places; tokens past the chunk's last repeat the
// last one with a step size of 0, which leaves the state as it is and gives the same output again.
// Other blocks (packed sequences' borders) go token by token.
template <typename T, int NP, bool PACKED, bool FAST, bool STATE_ONLY>
__global__ void __launch_bounds__(256) scan_fwd_kernel(ScanArgs p) {
  const Tile w(p);
  if (w.idle(p) || (STATE_ONLY && w.chunk + 1 == p.nch)) return;
  const int row = w.row;
  float A2[NP], h[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] = n < p.N ? p.A[(int64_t)w.d * p.N + n] * LOG2E_F : 0.f;
    h[n] = 0.f;
  }
  if (!STATE_ONLY && w.chunk > 0) load_slot<NP, FAST>(enter_slot(p, row, w.chunk), p, w.d, h);
  if (!PACKED && w.chunk == 0) entering_state<NP>(p, row, w.d, h);
  const float Dp = p.Dp ? p.Dp[w.d] : 0.f, bias = p.bias ? p.bias[w.d] : 0.f;
  const bool gated = p.z != nullptr, plus = p.softplus;
  const T* u = (const T*)p.u + row * p.u_sb;
  const T* dl = (const T*)p.delta + row * p.delta_sb;
  const T* z = gated ? (const T*)p.z + row * p.z_sb : u;        // (read and not used without z)
  const int64_t z_st = gated ? p.z_st : p.u_st;
  const T* B = (const T*)p.B + row * p.B_sb + w.g * p.B_sg;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  T* out = (T*)p.out + (int64_t)row * p.L * p.D;
  const uint32_t at = w.d * (uint32_t)sizeof(T);
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};
  if (PACKED) q.seek(w.t0);
  float total = 0.f;
  bool cut = false;
  FwdRaw<T> next;
  BCAhead<T, NP, FAST> ahead;
  const T *un = u + w.t0 * p.u_st, *dn = dl + w.t0 * p.delta_st, *zn = z + w.t0 * z_st;    // rows of the block ahead
  next.template load<!STATE_ONLY>(un, p.u_st, dn, p.delta_st, zn, z_st, w.t1 - w.t0, at);

  for (int t0 = w.t0; t0 < w.t1; t0 += SCAN_Q) {
    const int n = min(SCAN_Q, w.t1 - t0);
    const FwdRaw<T> raw = next;
    const int left = w.t1 - t0 - SCAN_Q;
    un += left > 0 ? p.u_st : 0;
    dn += left > 0 ? p.delta_st : 0;
    zn += left > 0 ? z_st : 0;
    next.template load<!STATE_ONLY>(un, p.u_st, dn, p.delta_st, zn, z_st, left, at);
    if (!STATE_ONLY && p.ckpt)
      store_slot<NP, FAST>(p.ckpt + ((int64_t)row * p.blocks + t0 / SCAN_Q) * p.N * p.D, p, w.d, h);
    Marks m = {0u, 0u, 0u};
    if (PACKED) m = block_marks<PACKED>(q, t0, n, p.L);
    if (!PACKED || !(m.start | m.end | (m.valid ^ ((1u << n) - 1u)))) {
      const T *Bt = B + t0 * p.B_st, *Ct = C + t0 * p.C_st;
      T* ot = out + (int64_t)t0 * p.D;
      if (STATE_ONLY) ahead.request_b(Bt, p.N);
      else ahead.request(Bt, Ct, p.N);
#pragma unroll
      for (int j = 0; j < SCAN_Q; ++j) {
        BCAhead<T, NP, FAST> now = ahead;
        float Bv[NP], Cv[NP];
        Bt += j + 1 < n ? p.B_st : 0;
        Ct += j + 1 < n ? p.C_st : 0;
        if (STATE_ONLY) {
          now.arrived_b(Bt);
          if (j + 1 < SCAN_Q) ahead.request_b(Bt, p.N);
          now.get_b(Bv);
        } else {
          now.arrived(Bt, Ct);
          if (j + 1 < SCAN_Q) ahead.request(Bt, Ct, p.N);
          now.get(Bv, Cv);
        }
        const float uu = to_f32(raw.u[j]);
        const float pre = to_f32(raw.dl[j]) + bias;
        const float sp = softplus_hw(pre);
        const float dt = j < n ? (plus ? sp : pre) : 0.f;
        const float x = dt * uu;
        if (STATE_ONLY) {
          total += dt;
#pragma unroll
          for (int i = 0; i < NP; ++i) h[i] = fmaf(exp2_hw(dt * A2[i]), h[i], x * Bv[i]);
        } else {
          float y = Dp * uu;
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            h[i] = fmaf(exp2_hw(dt * A2[i]), h[i], x * Bv[i]);
            y = fmaf(Cv[i], h[i], y);
          }
          const float zz = to_f32(raw.z[j]);
          const float gate = zz * sigmoid_hw(zz);
          lane_store(ot, at, from_f32<T>(gated ? y * gate : y));
          ot += j + 1 < n ? p.D : 0;
        }
      }
      continue;
    }
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int64_t t = t0 + j;
      if (!(m.valid >> j & 1)) {
        if (!STATE_ONLY) lane_store(out + t * p.D, at, from_f32<T>(0.f));
        continue;
      }
      if (m.start >> j & 1) {
        entering_state<NP>(p, q.seq(), w.d, h);
        cut = true;
      }
      const float uu = to_f32(lane_load(u + t * p.u_st, at));
      const float pre = to_f32(lane_load(dl + t * p.delta_st, at)) + bias;
      const float dt = plus ? softplus_hw(pre) : pre;
      float Bv[NP];
      BCLoad<T, NP, FAST>::get(B, t * p.B_st, p.N, Bv);
      const float x = dt * uu;
      if (STATE_ONLY) {
        total += dt;
#pragma unroll
        for (int i = 0; i < NP; ++i) h[i] = fmaf(exp2_hw(dt * A2[i]), h[i], x * Bv[i]);
      } else {
        float Cv[NP];
        BCLoad<T, NP, FAST>::get(C, t * p.C_st, p.N, Cv);
        float y = Dp * uu;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          h[i] = fmaf(exp2_hw(dt * A2[i]), h[i], x * Bv[i]);
          y = fmaf(Cv[i], h[i], y);
        }
        if (gated) {
          const float zz = to_f32(lane_load(z + t * z_st, at));
          y *= zz * sigmoid_hw(zz);
        }
        lane_store(out + t * p.D, at, from_f32<T>(y));
      }
      if (m.end >> j & 1) {
        if (!STATE_ONLY && p.state1 && w.on) store_state<NP>(p.state1, q.seq(), p, w.d, h);
        q.next((int)t + 1);
      }
    }
  }
  if (STATE_ONLY) {
    if (w.on) {
      store_slot<NP, FAST>(enter_slot(p, row, w.chunk + 1), p, w.d, h);
      p.sumdt[((int64_t)row * p.nch + w.chunk) * p.D + w.d] = total;
    }
    if (w.g == 0 && w.part == 0 && threadIdx.x == 0) p.keep[row * p.nch + w.chunk] = cut ? 0.f : 1.f;
  } else if (!PACKED && p.state1 && w.on && w.chunk + 1 == p.nch) {
    store_state<NP>(p.state1, row, p, w.d, h);
  }
}

// The states (or, BACK, the adjoints) that enter the chunks: x = decay * x + own, along the axis.  Where a sequence
// starts inside a chunk nothing of what enters it gets through.  A thread owns one state of one channel.
#define JOIN_AHEAD 8
template <bool BACK>
__global__ void __launch_bounds__(256) scan_join_kernel(ScanArgs p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t ND = (int64_t)p.N * p.D;
  if (i >= ND) return;
  const int row = blockIdx.y, d = (int)(i % p.D), n = (int)(i / p.D);
  const float A2 = p.A[(int64_t)d * p.N + n] * LOG2E_F;
  const float* sumdt = p.sumdt + (int64_t)row * p.nch * p.D + d;
  float x = 0.f;
  for (int k0 = 0; k0 + 1 < p.nch; k0 += JOIN_AHEAD) {
    float own[JOIN_AHEAD], dec[JOIN_AHEAD], keep[JOIN_AHEAD];
#pragma unroll
    for (int j = 0; j < JOIN_AHEAD; ++j) {
      const int k = min(k0 + j, p.nch - 2);
      const int c = BACK ? p.nch - 1 - k : k;              // the chunk that x passes through
      own[j] = (BACK ? leave_slot(p, row, c - 1) : enter_slot(p, row, c + 1))[i];
      dec[j] = sumdt[(int64_t)c * p.D];
      keep[j] = uniform_load(p.keep, (int64_t)row * p.nch + c);
    }
#pragma unroll
    for (int j = 0; j < JOIN_AHEAD; ++j) {
      const int k = k0 + j;
      if (k + 1 >= p.nch) break;
      const int c = BACK ? p.nch - 1 - k : k;
      x = keep[j] != 0.f ? fmaf(exp2_hw(dec[j] * A2), x, own[j]) : own[j];
      (BACK ? leave_slot(p, row, c - 1) : enter_slot(p, row, c + 1))[i] = x;
    }
  }
}

// The way back.  With g = dout silu(z), for a sequence's tokens from the last to the first:
//   dh[n]  = C[n] g + (a[n] dh[n] of the token behind)
//   dC[n] += g h[n]        dB[n] += dh[n] dt u          (sums over the group's channels)
//   w      = a[n] dh[n] (what goes on to the token before);  k = w h_before[n]
//   dA[n] += k dt          ddt += k A[n] + dh[n] B[n] u  du += dh[n] B[n] dt
// The states are computed again, SCAN_Q tokens at a time, from those that the forward pass kept.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
#define DPP_HALF_MIRROR 0x141
#define DPP_ROR8 0x128
#define DPP_XOR2 0x4e     // quad_perm [2,3,0,1]
#define DPP_XOR1 0xb1     // quad_perm [1,0,3,2]

// Sums of 2 * NP values over the 64 lanes, all at once: a step adds the two halves of the wave (then of a half, ...) and
// lets one half go on with one value, the other with another, so the number of values halves with the number of lanes
// that still hold parts of one.  The sum of value sum_index(lane) ends up in `lane`.
template <int M> struct WaveSums {
  static __device__ __forceinline__ float run(float (&v)[M], int lane) {
    // 32 lanes apart, then 16: the swaps exchange the upper half of one register with the lower half of the other
#pragma unroll
    for (int i = 0; i < M / 2; ++i) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + M / 2]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 4; ++i) {
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + M / 4]), false, false);
      v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 8; ++i) {
      const float a = lane & 8 ? v[i + M / 8] : v[i], b = lane & 8 ? v[i] : v[i + M / 8];
      v[i] = a + dpp<DPP_ROR8>(b);
    }
#pragma unroll
    for (int i = 0; i < M / 16; ++i) {
      const float a = lane & 4 ? v[i + M / 16] : v[i], b = lane & 4 ? v[i] : v[i + M / 16];
      v[i] = a + dpp<DPP_HALF_MIRROR>(b);
    }
    if (M == 32) {
      const float a = lane & 2 ? v[1] : v[0], b = lane & 2 ? v[0] : v[1];
      v[0] = a + dpp<DPP_XOR2>(b);
    } else {
      v[0] += dpp<DPP_XOR2>(v[0]);
    }
    return v[0] + dpp<DPP_XOR1>(v[0]);
  }
  static __device__ __forceinline__ int index(int lane) {
    return (lane & 32 ? M / 2 : 0) + (lane & 16 ? M / 4 : 0) + (lane & 8 ? M / 8 : 0) + (lane & 4 ? M / 16 : 0) +
           (M == 32 && lane & 2 ? 1 : 0);
  }
};

// What a block of tokens reads per channel on the way back, as stored; tokens past the chunk's last are the last one again.
template <typename T> struct BwdRaw {
  T u[SCAN_Q], dl[SCAN_Q], z[SCAN_Q], g[SCAN_Q];
  template <bool U>
  __device__ __forceinline__ void load(const T* up, int64_t u_st, const T* dp, int64_t d_st, const T* zp, int64_t z_st,
                                       const T* gp, int64_t g_st, int n, uint32_t at) {
#pragma unroll
    for (int j = 0; j < SCAN_Q; ++j) {
      if (U) u[j] = lane_load(up, at);
      dl[j] = lane_load(dp, at);
      z[j] = lane_load(zp, at);
      g[j] = lane_load(gp, at);
      const bool more = j + 1 < SCAN_Q && j + 1 < n;
      if (U) up += more ? u_st : 0;
      dp += more ? d_st : 0;
      zp += more ? z_st : 0;
      gp += more ? g_st : 0;
    }
  }
};

// The adjoint that leaves a chunk to the left if nothing enters it from the right: the sum of C[n] g of its tokens up to
// the first start of a sequence, each through the decays from the chunk's first token to its own.
template <typename T, int NP, bool PACKED, bool FAST>
__global__ void __launch_bounds__(256) scan_bwd_state_kernel(ScanArgs p) {
  const Tile w(p);
  if (w.idle(p) || w.chunk == 0) return;
  const int row = w.row;
  float A2[NP], x[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] = n < p.N ? p.A[(int64_t)w.d * p.N + n] * LOG2E_F : 0.f;
    x[n] = 0.f;
  }
  const float bias = p.bias ? p.bias[w.d] : 0.f;
  const bool gated = p.z != nullptr, plus = p.softplus;
  const T* dl = (const T*)p.delta + row * p.delta_sb;
  const T* go = (const T*)p.dout + row * p.dout_sb;
  const T* z = gated ? (const T*)p.z + row * p.z_sb : go;
  const int64_t z_st = gated ? p.z_st : p.dout_st;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  const uint32_t at = w.d * (uint32_t)sizeof(T);
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};
  if (PACKED) q.seek(w.t0);
  float total = 0.f;
  bool cut = false;
  BwdRaw<T> next;
  next.template load<false>(nullptr, 0, dl + w.t0 * p.delta_st, p.delta_st, z + w.t0 * z_st, z_st,
                            go + w.t0 * p.dout_st, p.dout_st, w.t1 - w.t0, at);
  for (int t0 = w.t0; t0 < w.t1 && !cut; t0 += SCAN_Q) {
    const int n = min(SCAN_Q, w.t1 - t0);
    const BwdRaw<T> raw = next;
    const int64_t tn = min(t0 + SCAN_Q, w.t1 - 1);
    next.template load<false>(nullptr, 0, dl + tn * p.delta_st, p.delta_st, z + tn * z_st, z_st, go + tn * p.dout_st,
                              p.dout_st, w.t1 - t0 - SCAN_Q, at);
    Marks m = {0u, 0u, 0u};
    if (PACKED) m = block_marks<PACKED>(q, t0, n, p.L);
    if (!PACKED || !(m.start | m.end | (m.valid ^ ((1u << n) - 1u)))) {
      BCAhead<T, NP, FAST> ahead;
      const T* Ct = C + t0 * p.C_st;
      ahead.request_b(Ct, p.N);
#pragma unroll
      for (int j = 0; j < SCAN_Q; ++j) {
        BCAhead<T, NP, FAST> now = ahead;
        float Cv[NP];
        Ct += j + 1 < n ? p.C_st : 0;
        now.arrived_b(Ct);
        if (j + 1 < SCAN_Q) ahead.request_b(Ct, p.N);
        now.get_b(Cv);
        const float pre = to_f32(raw.dl[j]) + bias;
        const float sp = softplus_hw(pre);
        total += j < n ? (plus ? sp : pre) : 0.f;
        const float zz = to_f32(raw.z[j]), gate = zz * sigmoid_hw(zz);
        float g = to_f32(raw.g[j]);
        g = j < n ? (gated ? g * gate : g) : 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), Cv[i] * g, x[i]);
      }
      continue;
    }
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int64_t t = t0 + j;
      if (!(m.valid >> j & 1)) continue;
      if (m.start >> j & 1) { cut = true; break; }
      const float pre = to_f32(lane_load(dl + t * p.delta_st, at)) + bias;
      total += plus ? softplus_hw(pre) : pre;
      float g = to_f32(lane_load(go + t * p.dout_st, at));
      if (gated) {
        const float zz = to_f32(lane_load(z + t * z_st, at));
        g *= zz * sigmoid_hw(zz);
      }
      float Cv[NP];
      BCLoad<T, NP, FAST>::get(C, t * p.C_st, p.N, Cv);
#pragma unroll
      for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), Cv[i] * g, x[i]);
      if (m.end >> j & 1) {
        if (p.dstate1) {
          float e[NP];
          load_state<NP>(p.dstate1, q.seq(), p, w.d, e);
#pragma unroll
          for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), e[i], x[i]);
        }
        q.next((int)t + 1);
      }
    }
  }
  if (!PACKED && p.dstate1 && w.chunk + 1 == p.nch) {
    float e[NP];
    load_state<NP>(p.dstate1, row, p, w.d, e);
#pragma unroll
    for (int i = 0; i < NP; ++i) x[i] = fmaf(exp2_hw(total * A2[i]), e[i], x[i]);
  }
  if (w.on) {
    store_slot<NP, FAST>(leave_slot(p, row, w.chunk - 1), p, w.d, x);
    p.sumdt[((int64_t)row * p.nch + w.chunk) * p.D + w.d] = total;
  }
  if (w.g == 0 && w.part == 0 && threadIdx.x == 0) p.keep[row * p.nch + w.chunk] = cut ? 0.f : 1.f;
}

template <typename T, int NP, bool PACKED, bool FAST>
__global__ void __launch_bounds__(256, 1) scan_bwd_kernel(ScanArgs p) {
  __shared__ float red[2][SCAN_Q][4][2 * NP];      // [block parity][token][wave][dB, dC]
  const Tile w(p);
  const int row = w.row;
  const bool idle = w.idle(p);                     // such a wave only takes part in the sums
  float A2[NP], dh[NP], dA[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] = n < p.N ? p.A[(int64_t)w.d * p.N + n] * LOG2E_F : 0.f;
    dh[n] = dA[n] = 0.f;
  }
  if (w.chunk + 1 < p.nch) load_slot<NP, FAST>(leave_slot(p, row, w.chunk), p, w.d, dh);
  else if (!PACKED && p.dstate1) load_state<NP>(p.dstate1, row, p, w.d, dh);
  float dD = 0.f, dbias = 0.f;
  const float Dp = p.Dp ? p.Dp[w.d] : 0.f, bias = p.bias ? p.bias[w.d] : 0.f;
  const T* u = (const T*)p.u + row * p.u_sb;
  const T* dl = (const T*)p.delta + row * p.delta_sb;
  const bool gated = p.z != nullptr, plus = p.softplus;
  const T* go = (const T*)p.dout + row * p.dout_sb;
  const T* z = gated ? (const T*)p.z + row * p.z_sb : go;             // (read and not used without z)
  const int64_t z_st = gated ? p.z_st : p.dout_st;
  T* dzp = gated ? (T*)p.dz : (T*)p.du;                                // (written and written over by du without z)
  const T* B = (const T*)p.B + row * p.B_sb + w.g * p.B_sg;
  const T* C = (const T*)p.C + row * p.C_sb + w.g * p.C_sg;
  const int64_t flat = (int64_t)row * p.L;
  const uint32_t at = w.d * (uint32_t)sizeof(T);
  SeqWalk q = {p.offsets, p.S, p.L, p.L, row, 0, p.L};      // the sequence that the way back is in
  if (PACKED) {                                             // the last one that has a token before the chunk's end
    q.seek(w.t1 - 1);
    if (q.s >= q.S || q.b >= w.t1) q.prev(w.t1 - 1);
  }
  int turn = 0;
  const int first = w.t0 + (w.t1 - w.t0 - 1) / SCAN_Q * SCAN_Q;
  const float* ck = p.ckpt + ((int64_t)row * p.blocks + first / SCAN_Q) * p.N * p.D;
  BwdRaw<T> next;
  float hn[NP];                                    // the state that enters the block ahead
  next.template load<true>(u + first * p.u_st, p.u_st, dl + first * p.delta_st, p.delta_st, z + first * z_st, z_st,
                           go + first * p.dout_st, p.dout_st, w.t1 - first, at);
  load_slot<NP, FAST>(ck, p, w.d, hn);

  for (int t0 = first; t0 >= w.t0; t0 -= SCAN_Q, turn ^= 1) {
    const int n = min(SCAN_Q, w.t1 - t0);
    const BwdRaw<T> raw = next;
    float hs[SCAN_Q + 1][NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) hs[0][i] = hn[i];
    {
      const int64_t tn = max(t0 - SCAN_Q, w.t0);
      ck -= t0 > w.t0 ? (int64_t)p.N * p.D : 0;
      next.template load<true>(u + tn * p.u_st, p.u_st, dl + tn * p.delta_st, p.delta_st, z + tn * z_st, z_st,
                               go + tn * p.dout_st, p.dout_st, w.t1 - tn, at);
      load_slot<NP, FAST>(ck, p, w.d, hn);
    }
    SeqWalk f = q;                                 // the sequence that the states' second computation is in
    Marks m = {0u, 0u, 0u};
    if (PACKED) {
      f.seek(t0);
      m = block_marks<PACKED>(f, t0, n, p.L);
    }
    if (idle) {
      for (int i = w.lane; i < SCAN_Q * 2 * NP; i += 64) red[turn][i / (2 * NP)][w.wave][i % (2 * NP)] = 0.f;
    } else if (!PACKED || !(m.start | m.end | (m.valid ^ ((1u << n) - 1u)))) {
      // no sequence starts or ends here: straight-line code, as in the forward pass.  Tokens past the chunk's last have
      // a step size and a gradient of 0, which changes nothing, and what they store is stored over by the last token.
      float a[SCAN_Q][NP], db[SCAN_Q], slope[SCAN_Q];
      BCAhead<T, NP, FAST> ahead;
      const T *Bt = B + t0 * p.B_st, *Ct = C + t0 * p.C_st;
      ahead.request_b(Bt, p.N);
#pragma unroll
      for (int j = 0; j < SCAN_Q; ++j) {
        BCAhead<T, NP, FAST> now = ahead;
        float Bv[NP];
        Bt += j + 1 < n ? p.B_st : 0;
        Ct += j + 1 < n ? p.C_st : 0;
        now.arrived_b(Bt);
        if (j + 1 < SCAN_Q) ahead.request_b(Bt, p.N);
        else ahead.request(Bt, Ct, p.N);           // the last token's, where the way back begins
        now.get_b(Bv);
        const float pre = to_f32(raw.dl[j]) + bias;
        const float sp = softplus_hw(pre, slope[j]);
        db[j] = j < n ? (plus ? sp : pre) : 0.f;
        slope[j] = plus ? slope[j] : 1.f;
        const float x = db[j] * to_f32(raw.u[j]);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          a[j][i] = exp2_hw(db[j] * A2[i]);
          hs[j + 1][i] = fmaf(a[j][i], hs[j][i], x * Bv[i]);
        }
      }
      int64_t o = (flat + t0 + n - 1) * p.D;
#pragma unroll
      for (int j = SCAN_Q - 1; j >= 0; --j) {
        BCAhead<T, NP, FAST> now = ahead;
        float Bv[NP], Cv[NP];
        Bt -= j > 0 && j < n ? p.B_st : 0;
        Ct -= j > 0 && j < n ? p.C_st : 0;
        now.arrived(Bt, Ct);
        if (j > 0) ahead.request(Bt, Ct, p.N);
        now.get(Bv, Cv);
        const float uu = to_f32(raw.u[j]), zz = to_f32(raw.z[j]), sg = sigmoid_hw(zz);
        float g = j < n ? to_f32(raw.g[j]) : 0.f;
        float y = Dp * uu;
#pragma unroll
        for (int i = 0; i < NP; ++i) y = fmaf(Cv[i], hs[j + 1][i], y);
        lane_store(dzp + o, at, from_f32<T>(g * y * sg * fmaf(zz, 1.f - sg, 1.f)));
        g = gated ? g * (zz * sg) : g;
        // lanes past the last channel add nothing to the sums over the channels
        const float x = w.on ? db[j] * uu : 0.f, gs = w.on ? g : 0.f;
        float through = 0.f, ka = 0.f, pv[2 * NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float d = fmaf(Cv[i], g, dh[i]);
          pv[i] = d * x;
          pv[NP + i] = gs * hs[j + 1][i];
          through = fmaf(d, Bv[i], through);
          dh[i] = d * a[j][i];
          const float k = dh[i] * hs[j][i];
          dA[i] = fmaf(k, db[j], dA[i]);
          ka = fmaf(k, A2[i], ka);
        }
        const float sum = WaveSums<2 * NP>::run(pv, w.lane);
        if (!(w.lane & (NP == 16 ? 1 : 3))) red[turn][j][w.wave][WaveSums<2 * NP>::index(w.lane)] = sum;
        dD = fmaf(g, uu, dD);
        float dd = fmaf(ka, LN2_F, through * uu) * slope[j];
        dd = j < n ? dd : 0.f;
        dbias += dd;
        lane_store((T*)p.du + o, at, from_f32<T>(fmaf(through, db[j], Dp * g)));
        lane_store((T*)p.ddelta + o, at, from_f32<T>(dd));
        o -= j < n ? p.D : 0;
      }
    } else {
      float ub[SCAN_Q], pb[SCAN_Q], db[SCAN_Q];
#pragma unroll
      for (int j = 0; j < SCAN_Q; ++j) {
#pragma unroll
        for (int i = 0; i < NP; ++i) hs[j + 1][i] = hs[j][i];
        if (!(m.valid >> j & 1)) continue;
        const int64_t t = t0 + j;
        ub[j] = to_f32(raw.u[j]);
        pb[j] = to_f32(raw.dl[j]) + bias;
        db[j] = plus ? softplus_hw(pb[j]) : pb[j];
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
            if (gated) ((T*)p.dz)[o] = from_f32<T>(0.f);
          }
          if (w.lane < 2 * NP) red[turn][j][w.wave][w.lane] = 0.f;
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
        float g = to_f32(raw.g[j]);
        if (gated) {
          const float zz = to_f32(raw.z[j]);
          const float sg = sigmoid_hw(zz);
          float y = Dp * ub[j];
#pragma unroll
          for (int i = 0; i < NP; ++i) y = fmaf(Cv[i], hs[j + 1][i], y);
          if (w.on) ((T*)p.dz)[o] = from_f32<T>(g * y * sg * fmaf(zz, 1.f - sg, 1.f));
          g *= zz * sg;
        }
        const float x = w.on ? db[j] * ub[j] : 0.f, gs = w.on ? g : 0.f;
        float through = 0.f, ka = 0.f, pv[2 * NP], hb[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) hb[i] = hs[j][i];
        if (m.start >> j & 1) entering_state<NP>(p, q.seq(), w.d, hb);
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const float a = exp2_hw(db[j] * A2[i]);
          const float d = fmaf(Cv[i], g, dh[i]);
          pv[i] = d * x;
          pv[NP + i] = gs * hs[j + 1][i];
          through = fmaf(d, Bv[i], through);
          dh[i] = d * a;
          const float k = dh[i] * hb[i];
          dA[i] = fmaf(k, db[j], dA[i]);
          ka = fmaf(k, A2[i], ka);
        }
        const float sum = WaveSums<2 * NP>::run(pv, w.lane);
        if (!(w.lane & (NP == 16 ? 1 : 3))) red[turn][j][w.wave][WaveSums<2 * NP>::index(w.lane)] = sum;
        dD = fmaf(g, ub[j], dD);
        float dd = fmaf(ka, LN2_F, through * ub[j]);
        if (plus) dd *= sigmoid_hw(pb[j]);
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
    __syncthreads();           // the other parity's buffer was read before the last of these, so one barrier is enough
    for (int i = threadIdx.x; i < n * 2 * p.N; i += 256) {
      const int j = i / (2 * p.N), c = i % (2 * p.N), k = c < p.N ? c : c - p.N + NP;
      const float s = (red[turn][j][0][k] + red[turn][j][1][k]) + (red[turn][j][2][k] + red[turn][j][3][k]);
      p.part_bc[(((int64_t)w.part * p.rows * p.L + flat + t0 + j) * p.G + w.g) * 2 * p.N + c] = s;
    }
  }
  if (!PACKED && w.chunk == 0 && p.dstate0 && w.on && !idle) store_state<NP>(p.dstate0, row, p, w.d, dh);
  if (w.on && !idle) {
    float* pa = p.part_a + ((int64_t)row * p.nch + w.chunk) * (p.N + 2) * p.D + w.d;
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

// dA [D][N], dD [D], dbias [D] from the partial rows [parts][N + 2][D]
__global__ void __launch_bounds__(64 * SUM_WAVES) scan_params_kernel(const float* part, float* dA, float* dD, float* dbias,
                                                                     int parts, int N, int D) {
  const int64_t total = (int64_t)(N + 2) * D;
  const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float s = column_sum(part, parts, total, i, i < total);
  if (threadIdx.x >= 64 || i >= total) return;
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
  p.wpg = p.G * ((p.tpg + 3) / 4);
  p.blocks = (int)ceil_div64(L, SCAN_Q);
  // as many chunks as it takes to reach SCAN_WAVES waves, none shorter than SCAN_MIN_CHUNK tokens
  const int64_t waves = rows * p.tpg * G;
  int64_t n = waves > 0 ? ceil_div64(SCAN_WAVES, waves) : 1;
  const int64_t most = L / SCAN_MIN_CHUNK;
  n = n < most ? n : most;
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

// whether B and C of every token and group can be read as whole aligned words
static bool scan_words(const ScanArgs& p, int dtype, int NP) {
  if (p.N != NP) return false;
  if (dtype == DVAE_DT_F32) return true;
  const int64_t odd = p.B_sb | p.B_st | p.B_sg | p.C_sb | p.C_st | p.C_sg;
  return !(odd & 1) && !(((uintptr_t)p.B | (uintptr_t)p.C) & 3);
}

template <typename T, int NP, bool PACKED, bool FAST> static void scan_fwd_launch(const ScanArgs& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.rows * p.nch * p.wpg)), block(256);
  if (p.nch > 1) {
    DVAE_LAUNCH((scan_fwd_kernel<T, NP, PACKED, FAST, true>), grid, block, 0, s, p);
    DVAE_LAUNCH((scan_join_kernel<false>), dim3((unsigned)ceil_div64((int64_t)p.N * p.D, 256), p.rows), block, 0, s, p);
  }
  DVAE_LAUNCH((scan_fwd_kernel<T, NP, PACKED, FAST, false>), grid, block, 0, s, p);
}
template <typename T, int NP, bool PACKED, bool FAST> static void scan_bwd_launch(const ScanArgs& p, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)p.rows * p.nch * p.wpg)), block(256);
  if (p.nch > 1) {
    DVAE_LAUNCH((scan_bwd_state_kernel<T, NP, PACKED, FAST>), grid, block, 0, s, p);
    DVAE_LAUNCH((scan_join_kernel<true>), dim3((unsigned)ceil_div64((int64_t)p.N * p.D, 256), p.rows), block, 0, s, p);
  }
  DVAE_LAUNCH((scan_bwd_kernel<T, NP, PACKED, FAST>), grid, block, 0, s, p);
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
  const int64_t parts = (p.tpg + 3) / 4, chunks = rows * p.nch;
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
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.u_st = u_st; p.delta = delta; p.delta_sb = delta_sb; p.delta_st = delta_st; p.A = A;
  p.B = B; p.B_sb = B_sb; p.B_st = B_st; p.B_sg = B_sg; p.C = C; p.C_sb = C_sb; p.C_st = C_st; p.C_sg = C_sg;
  p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.z_st = z_st; p.bias = bias; p.softplus = softplus;
  p.state0 = state0; p.state1 = state1; p.offsets = offsets; p.out = out; p.ckpt = ckpt;
  scan_shape(p, rows, L, D, G, N, S);
  scan_scratch(p, ws);
  DVAE_REQUIRE(rows * p.nch * p.wpg < (1ll << 31), "selective_scan_fwd: too many rows");
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
  DVAE_REQUIRE(!z || dz, "selective_scan_bwd: dz is needed with z");
  ScanArgs p = {};
  p.u = u; p.u_sb = u_sb; p.u_st = u_st; p.delta = delta; p.delta_sb = delta_sb; p.delta_st = delta_st; p.A = A;
  p.B = B; p.B_sb = B_sb; p.B_st = B_st; p.B_sg = B_sg; p.C = C; p.C_sb = C_sb; p.C_st = C_st; p.C_sg = C_sg;
  p.Dp = Dp; p.z = z; p.z_sb = z_sb; p.z_st = z_st; p.bias = bias; p.softplus = softplus;
  p.state0 = state0; p.offsets = offsets; p.dout = dout; p.dout_sb = dout_sb; p.dout_st = dout_st;
  p.dstate1 = dstate1; p.dstate0 = dstate0; p.ckpt = const_cast<float*>(ckpt);
  p.du = du; p.ddelta = ddelta; p.dz = dz;
  scan_shape(p, rows, L, D, G, N, S);
  const int parts = (p.tpg + 3) / 4;
  float* after = scan_scratch(p, ws);
  if (p.nch == 1) after = ws;
  else { p.leave = after; after += (int64_t)rows * p.nch * N * D; }
  p.part_bc = after;
  p.part_a = after + (int64_t)parts * rows * L * G * 2 * N;
  DVAE_REQUIRE(rows * p.nch * p.wpg < (1ll << 31), "selective_scan_bwd: too many rows");
  const int e = dtype == DVAE_DT_F32 ? 4 : 2;
  DVAE_WORK(rows * L * (double)e * ((z ? 7 : 5) * D + 4 * G * N), DVAE_UNIT_BYTE);
  SCAN_DISPATCH(scan_bwd_launch, dtype, p, ST(stream));
  DVAE_LAUNCH_CHECK("selective_scan_bwd");
  const int64_t bc = rows * L * G;
  const dim3 gbc((unsigned)ceil_div64(bc * 2 * N, 256));
  if (dtype == DVAE_DT_F32)
    DVAE_LAUNCH((scan_bc_kernel<float>), gbc, dim3(256), 0, ST(stream), p.part_bc, (float*)dB, (float*)dC, bc, p.N, parts);
  else
    DVAE_LAUNCH((scan_bc_kernel<bf16_t>), gbc, dim3(256), 0, ST(stream), p.part_bc, (bf16_t*)dB, (bf16_t*)dC, bc, p.N, parts);
  DVAE_LAUNCH(scan_params_kernel, dim3((unsigned)ceil_div64((int64_t)(p.N + 2) * D, 64)), dim3(64 * SUM_WAVES), 0, ST(stream),
              p.part_a, dA, dD, dbias, p.rows * p.nch, p.N, p.D);
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
