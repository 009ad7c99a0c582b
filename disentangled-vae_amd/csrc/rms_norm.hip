// Root-mean-square norm with the residual's addition: sum = x + residual (rounded to its stored type),
// y = sum * rstd * w with rstd = 1 / sqrt(mean(sum^2) + eps).  The norm is that of the stored sum, so the backward pass,
// which reads the sum again, works on the very numbers that the forward pass normalised.  Squares are added in fp32.
//
// Bound by memory.  A wave owns a row and holds it in registers between the reduction and the output (up to 64 values
// per lane: rows of up to 4096 elements whose tensors are 16-byte aligned), so every tensor crosses memory once and no
// barrier is needed.  Longer or unaligned rows take one workgroup each, which goes element by element and reads its row a
// second time, and dw is a pass of its own.
//
// 16384 x 2048 bf16: forward 57 us (4.7 TB/s of x, residual, sum and y), backward 65 us (4.1 TB/s of dy, dsum, sum and
// dresidual) and 4 us for the sums of its partial rows; with an fp32 residual 85 us (4.7 TB/s) and 112 us (4.8 TB/s); 4099 x
// 2560 bf16 into 8 bits: 18 us (4.1 TB/s).  A copy of 2 GiB runs at 4.9 TB/s on the same card.  Rows of the second kind:
// 4096 x 8192 bf16 forward 101 us (2.7 TB/s), backward 109 and 28 for dw; 16384 x 2047 bf16 113, 109 and 30 us.
#include "seq_common.h"

struct NormArgs {
  const void *x, *res, *dy, *dsum, *sum_in;
  int64_t x_st, r_st, dy_st, ds_st, s_st;
  const float* w;
  const float* rstd_in;
  float eps;
  void *y, *sum, *dres, *dx;
  float *rstd, *scale, *part;
  int64_t rows;
  int D;
};

#define FP8_MAX 448.f

__device__ __forceinline__ uint32_t fp8_pair(float a, float b) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
template <int V>
__device__ __forceinline__ void store_fp8(uint8_t* p, const float (&v)[V]) {
  if (V == 1) {
    *p = (uint8_t)fp8_pair(v[0], v[0]);
  } else {
    Pack<uint32_t, V / 4 ? V / 4 : 1> r;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) r.v[i] = fp8_pair(v[4 * i], v[4 * i + 1]) | fp8_pair(v[4 * i + 2], v[4 * i + 3]) << 16;
    *reinterpret_cast<Pack<uint32_t, V / 4 ? V / 4 : 1>*>(p) = r;
  }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o);
    v = u > v || u != u ? u : v;               // NaN stays
  }
  return v;
}
__device__ __forceinline__ float max_abs(float m, float v) {
  v = fabsf(v);
  return v > m || v != v ? v : m;
}

// The scale of a row whose largest value is `most`, not below the smallest normal number: a scale of fewer bits would be
// rounded by so much that the largest value comes out behind the type's end.
__device__ __forceinline__ float row_scale(float most) {
  const float s = most / FP8_MAX;
  return most == 0.f ? 1.f : s < __FLT_MIN__ ? __FLT_MIN__ : s;
}

template <typename T, typename R>
__device__ __forceinline__ float rounded_sum(float x, float r) { return to_f32(from_f32<R>(x + r)); }

template <typename T, typename R, int V, int NV, bool Q8>
__global__ void __launch_bounds__(256) norm_row_kernel(NormArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  float v[NV][V];
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int d = (k * 64 + lane) * V;
    if (d < p.D) {
      load_pack<T, V>((const T*)p.x + row * p.x_st + d, v[k]);
      if (p.res) {
        float r[V];
        load_pack<R, V>((const R*)p.res + row * p.r_st + d, r);
#pragma unroll
        for (int i = 0; i < V; ++i) v[k][i] = rounded_sum<T, R>(v[k][i], r[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sq = fmaf(v[k][i], v[k][i], sq);
  }
  const float rstd = 1.f / sqrtf(wave_sum(sq) / p.D + p.eps);
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int d = (k * 64 + lane) * V;
    if (d < p.D) {
      if (p.res) store_pack<R, V>((R*)p.sum + row * p.D + d, v[k]);
      float w[V];
      load_pack<float, V>(p.w + d, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] = v[k][i] * rstd * w[i];
        if (Q8) most = max_abs(most, v[k][i]);
      }
      if (!Q8) store_pack<T, V>((T*)p.y + row * p.D + d, v[k]);
    }
  }
  if (!Q8) {
    if (p.rstd && lane == 0) p.rstd[row] = rstd;
    return;
  }
  most = wave_max(most);
  const float scale = row_scale(most);
  if (lane == 0) p.scale[row] = scale;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int d = (k * 64 + lane) * V;
    if (d < p.D) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = v[k][i] / scale;
      store_fp8<V>((uint8_t*)p.y + row * p.D + d, v[k]);
    }
  }
}

// sum over the workgroup's four waves, the same in every thread
__device__ __forceinline__ float block_sum4(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// any row: one workgroup, element by element, the row read again for the output (out of the L2)
template <typename T, typename R, bool Q8>
__global__ void __launch_bounds__(256) norm_any_kernel(NormArgs p) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.x + row * p.x_st;
  const R* r = p.res ? (const R*)p.res + row * p.r_st : nullptr;
  float sq = 0.f;
  for (int d = threadIdx.x; d < p.D; d += 256) {
    const float v = r ? rounded_sum<T, R>(to_f32(x[d]), to_f32(r[d])) : to_f32(x[d]);
    sq = fmaf(v, v, sq);
  }
  const float rstd = 1.f / sqrtf(block_sum4(sq, red) / p.D + p.eps);
  float most = 0.f;
  for (int d = threadIdx.x; d < p.D; d += 256) {
    const float v = r ? rounded_sum<T, R>(to_f32(x[d]), to_f32(r[d])) : to_f32(x[d]);
    if (r) ((R*)p.sum)[row * p.D + d] = from_f32<R>(v);
    if (Q8) most = max_abs(most, v * rstd * p.w[d]);
    else ((T*)p.y)[row * p.D + d] = from_f32<T>(v * rstd * p.w[d]);
  }
  if (!Q8) {
    if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
    return;
  }
  most = wave_max(most);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
  __syncthreads();
  most = max_abs(max_abs(max_abs(red[0], red[1]), red[2]), red[3]);
  const float scale = row_scale(most);
  if (threadIdx.x == 0) p.scale[row] = scale;
  for (int d = threadIdx.x; d < p.D; d += 256) {
    const float v = r ? rounded_sum<T, R>(to_f32(x[d]), to_f32(r[d])) : to_f32(x[d]);
    ((uint8_t*)p.y)[row * p.D + d] = (uint8_t)fp8_pair(v * rstd * p.w[d] / scale, 0.f);
  }
}

// With hat = sum * rstd and gw = w dy: dv = rstd (gw - hat mean(gw hat)) + dsum, dw = sum over rows of dy hat.  A wave
// takes every gridDim*4-th row and keeps its share of dw in registers until the end.
template <typename T, typename R, int V, int NV>
__global__ void __launch_bounds__(256) norm_bwd_row_kernel(NormArgs p) {
  extern __shared__ float red[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float dw[NV][V] = {};
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < p.rows; row += (int64_t)gridDim.x * 4) {
    float hat[NV][V], gw[NV][V], c = 0.f;
    const float rstd = p.rstd_in[row];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int d = (k * 64 + lane) * V;
      if (d < p.D) {
        load_pack<R, V>((const R*)p.sum_in + row * p.s_st + d, hat[k]);
        load_pack<T, V>((const T*)p.dy + row * p.dy_st + d, gw[k]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) hat[k][i] = gw[k][i] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int d = (k * 64 + lane) * V;
      float w[V] = {};
      if (d < p.D) load_pack<float, V>(p.w + d, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        hat[k][i] *= rstd;
        dw[k][i] = fmaf(gw[k][i], hat[k][i], dw[k][i]);
        gw[k][i] *= w[i];
        c = fmaf(gw[k][i], hat[k][i], c);
      }
    }
    c = wave_sum(c) / p.D;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int d = (k * 64 + lane) * V;
      if (d >= p.D) continue;
      float o[V] = {};
      if (p.dsum) load_pack<R, V>((const R*)p.dsum + row * p.ds_st + d, o);
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(rstd, fmaf(-hat[k][i], c, gw[k][i]), o[i]);
      store_pack<R, V>((R*)p.dres + row * p.D + d, o);
      if (p.dx) store_pack<T, V>((T*)p.dx + row * p.D + d, o);
    }
  }
  for (int turn = 0; turn < 4; ++turn) {
    if (wave == turn) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int j = (k * V + i) * 64 + lane;
          red[j] = turn ? red[j] + dw[k][i] : dw[k][i];
        }
    }
    __syncthreads();
  }
  for (int j = threadIdx.x; j < NV * V * 64; j += 256) {
    const int i = j / 64, d = ((i / V) * 64 + j % 64) * V + i % V;
    if (d < p.D) p.part[(int64_t)blockIdx.x * p.D + d] = red[j];
  }
}

// any row: one workgroup, as in the forward pass; dw comes from a pass of its own, column by column
template <typename T, typename R>
__global__ void __launch_bounds__(256) norm_bwd_any_kernel(NormArgs p) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const R* s = (const R*)p.sum_in + row * p.s_st;
  const T* dy = (const T*)p.dy + row * p.dy_st;
  const float rstd = p.rstd_in[row];
  float c = 0.f;
  for (int d = threadIdx.x; d < p.D; d += 256) c = fmaf(to_f32(dy[d]) * p.w[d], to_f32(s[d]) * rstd, c);
  c = block_sum4(c, red) / p.D;
  for (int d = threadIdx.x; d < p.D; d += 256) {
    const float hat = to_f32(s[d]) * rstd;
    float o = p.dsum ? to_f32(((const R*)p.dsum)[row * p.ds_st + d]) : 0.f;
    o = fmaf(rstd, fmaf(-hat, c, to_f32(dy[d]) * p.w[d]), o);
    ((R*)p.dres)[row * p.D + d] = from_f32<R>(o);
    if (p.dx) ((T*)p.dx)[row * p.D + d] = from_f32<T>(o);
  }
}

#define NORM_DW_ROWS 64
template <typename T, typename R>
__global__ void __launch_bounds__(256) norm_dw_any_kernel(NormArgs p, int tiles) {
  const int d = (int)(blockIdx.x % tiles) * 256 + threadIdx.x;
  const int64_t part = blockIdx.x / tiles;
  if (d >= p.D) return;
  float a = 0.f;
  const int64_t end = min(p.rows, (part + 1) * NORM_DW_ROWS);
  for (int64_t r = part * NORM_DW_ROWS; r < end; ++r)
    a = fmaf(to_f32(((const T*)p.dy)[r * p.dy_st + d]), to_f32(((const R*)p.sum_in)[r * p.s_st + d]) * p.rstd_in[r], a);
  p.part[part * p.D + d] = a;
}

__global__ void __launch_bounds__(64 * SUM_WAVES) norm_dw_sum_kernel(const float* part, float* dw, int64_t parts, int D) {
  const int d = blockIdx.x * 64 + (threadIdx.x & 63);
  const float s = column_sum(part, parts, D, d, d < D);
  if (threadIdx.x < 64 && d < D) dw[d] = s;
}

// ------------------------------------------------------------------------------------------------ host side
#define NORM_MAX_GRID 512     // workgroups of the backward kernel, and with that partial rows of dw: two per compute unit
static int64_t norm_row_grid(int64_t rows) {
  const int64_t g = ceil_div64(rows, 4);
  return g < NORM_MAX_GRID ? g : NORM_MAX_GRID;
}

static int norm_check(const char* what, int64_t rows, int64_t D, int dtype, int rdtype) {
  DVAE_REQUIRE(dtype == DVAE_DT_F32 || dtype == DVAE_DT_BF16, "%s: dtype must be fp32 (0) or bf16 (1)", what);
  DVAE_REQUIRE(rdtype == dtype || rdtype == DVAE_DT_F32, "%s: the residual's type must be that of x, or fp32", what);
  DVAE_REQUIRE(rows >= 0 && rows < (1ll << 31) - 1 && D > 0 && D < (1ll << 24), "%s: bad shape", what);
  return 0;
}

// values per lane and access, 0 where the row does not fit the one-wave kernels
static int norm_v(int64_t D, int dtype, int64_t strides, uintptr_t ptrs) {
  const int V = dtype == DVAE_DT_F32 ? 4 : 8;
  return (ptrs & 15) || ((D | strides) & (V - 1)) || D > 4096 ? 0 : V;
}

// A launch holds fewer than 2^32 threads, so a call of very many rows takes several, of this many rows each.
static int64_t norm_span(int V) { return V ? 1ll << 25 : 1ll << 23; }
// the arguments of `n` rows from row r0 on; e, re, ye: bytes per element of x, residual and y
static NormArgs norm_rows(const NormArgs& p, int64_t r0, int64_t n, int e, int re, int ye) {
  NormArgs q = p;
  auto in = [&](const void* a, int64_t st, int size) { return a ? (const char*)a + r0 * st * size : nullptr; };
  auto out = [&](void* a, int64_t st, int size) { return a ? (char*)a + r0 * st * size : nullptr; };
  q.x = in(p.x, p.x_st, e); q.res = in(p.res, p.r_st, re); q.dy = in(p.dy, p.dy_st, e); q.dsum = in(p.dsum, p.ds_st, re);
  q.sum_in = in(p.sum_in, p.s_st, re); q.rstd_in = (const float*)in(p.rstd_in, 1, 4);
  q.y = out(p.y, p.D, ye); q.sum = out(p.sum, p.D, re); q.dres = out(p.dres, p.D, re); q.dx = out(p.dx, p.D, e);
  q.rstd = (float*)out(p.rstd, 1, 4); q.scale = (float*)out(p.scale, 1, 4);
  q.rows = n;
  return q;
}

#define NORM_NV(K, T, R, V, nv, ...)                                              \
  do {                                                                            \
    if (nv <= 1) K(T, R, V, 1, __VA_ARGS__);                                      \
    else if (nv <= 2) K(T, R, V, 2, __VA_ARGS__);                                 \
    else if (nv <= 4) K(T, R, V, 4, __VA_ARGS__);                                 \
    else if (nv <= 8) K(T, R, V, 8, __VA_ARGS__);                                 \
    else K(T, R, V, (V == 4 ? 16 : 8), __VA_ARGS__);                              \
  } while (0)
#define NORM_TYPES(DO)                                                            \
  do {                                                                            \
    if (dtype == DVAE_DT_F32) DO(float, float, 4);                                \
    else if (rdtype == DVAE_DT_BF16) DO(bf16_t, bf16_t, 8);                       \
    else DO(bf16_t, float, 8);                                                    \
  } while (0)

static int norm_fwd(const char* what, bool q8, const NormArgs& all, int dtype, int rdtype, hipStream_t s) {
  if (all.rows == 0) return 0;
  const int V = norm_v(all.D, dtype, all.x_st | (all.res ? all.r_st : 0),
                       (uintptr_t)all.x | (uintptr_t)all.res | (uintptr_t)all.w | (uintptr_t)all.y | (uintptr_t)all.sum);
  const int nv = V ? (int)ceil_div64(all.D, 64 * V) : 0;
  const int e = dtype == DVAE_DT_F32 ? 4 : 2, re = rdtype == DVAE_DT_F32 ? 4 : 2;
  const int64_t span = norm_span(V);
  for (int64_t r0 = 0; r0 < all.rows; r0 += span) {
    const NormArgs p = norm_rows(all, r0, all.rows - r0 < span ? all.rows - r0 : span, e, re, q8 ? 1 : e);
    const dim3 grid((unsigned)(V ? ceil_div64(p.rows, 4) : p.rows));
    DVAE_WORK((double)p.rows * p.D * e * (p.res ? 4 : 2), DVAE_UNIT_BYTE);
#define NORM_ROW(T, R, V, NV, q) DVAE_LAUNCH((norm_row_kernel<T, R, V, NV, q>), grid, dim3(256), 0, s, p)
#define NORM_FWD(T, R, VV)                                                              \
  do {                                                                                  \
    if (V && q8) NORM_NV(NORM_ROW, T, R, VV, nv, true);                                 \
    else if (V) NORM_NV(NORM_ROW, T, R, VV, nv, false);                                 \
    else if (q8) DVAE_LAUNCH((norm_any_kernel<T, R, true>), grid, dim3(256), 0, s, p);  \
    else DVAE_LAUNCH((norm_any_kernel<T, R, false>), grid, dim3(256), 0, s, p);         \
  } while (0)
    NORM_TYPES(NORM_FWD);
  }
  DVAE_LAUNCH_CHECK(what);
  return 0;
}

extern "C" int dvae_add_rms_norm_fwd(const void* x, int64_t x_st, const void* residual, int64_t r_st, const float* w,
                                     float eps, void* y, void* sum, float* rstd, int64_t rows, int64_t D, int dtype,
                                     int rdtype, dvae_stream_t stream) {
  const int rc = norm_check("add_rms_norm_fwd", rows, D, dtype, rdtype);
  if (rc) return rc;
  NormArgs p = {};
  p.x = x; p.x_st = x_st; p.res = residual; p.r_st = r_st; p.w = w; p.eps = eps; p.y = y; p.sum = sum; p.rstd = rstd;
  p.rows = rows; p.D = (int)D;
  return norm_fwd("add_rms_norm_fwd", false, p, dtype, rdtype, ST(stream));
}

extern "C" int dvae_add_rms_norm_q8(const void* x, int64_t x_st, const void* residual, int64_t r_st, const float* w,
                                    float eps, void* q, float* scale, void* sum, int64_t rows, int64_t D, int dtype,
                                    int rdtype, dvae_stream_t stream) {
  const int rc = norm_check("add_rms_norm_q8", rows, D, dtype, rdtype);
  if (rc) return rc;
  NormArgs p = {};
  p.x = x; p.x_st = x_st; p.res = residual; p.r_st = r_st; p.w = w; p.eps = eps; p.y = q; p.sum = sum; p.scale = scale;
  p.rows = rows; p.D = (int)D;
  return norm_fwd("add_rms_norm_q8", true, p, dtype, rdtype, ST(stream));
}

extern "C" int64_t dvae_add_rms_norm_bwd_ws_floats(int64_t rows, int64_t D) {
  const int64_t a = norm_row_grid(rows), b = ceil_div64(rows, NORM_DW_ROWS);
  return (a > b ? a : b) * D;
}

extern "C" int dvae_add_rms_norm_bwd(const void* dy, int64_t dy_st, const void* dsum, int64_t ds_st, const void* sum,
                                     int64_t s_st, const float* w, const float* rstd, void* dres, void* dx, float* dw,
                                     int64_t rows, int64_t D, int dtype, int rdtype, float* ws, dvae_stream_t stream) {
  const int rc = norm_check("add_rms_norm_bwd", rows, D, dtype, rdtype);
  if (rc) return rc;
  DVAE_REQUIRE(rows > 0, "add_rms_norm_bwd: no rows");
  NormArgs p = {};
  p.dy = dy; p.dy_st = dy_st; p.dsum = dsum; p.ds_st = ds_st; p.sum_in = sum; p.s_st = s_st; p.w = w; p.rstd_in = rstd;
  p.dres = dres; p.dx = dtype == rdtype ? nullptr : dx; p.part = ws; p.rows = rows; p.D = (int)D;
  const hipStream_t s = ST(stream);
  const int V = norm_v(D, dtype, dy_st | s_st | (dsum ? ds_st : 0),
                       (uintptr_t)dy | (uintptr_t)dsum | (uintptr_t)sum | (uintptr_t)w | (uintptr_t)dres | (uintptr_t)p.dx);
  DVAE_WORK((double)rows * D * (dtype == DVAE_DT_F32 ? 4 : 2) * 4, DVAE_UNIT_BYTE);
  int64_t parts;
  if (V) {
    parts = norm_row_grid(rows);
    const dim3 grid((unsigned)parts);
    const int nv = (int)ceil_div64(D, 64 * V);
#define NORM_BWD_ROW(T, R, V, NV, s)                                                                       \
  DVAE_LAUNCH((norm_bwd_row_kernel<T, R, V, NV>), grid, dim3(256), NV * V * 64 * sizeof(float), s, p)
#define NORM_BWD(T, R, VV) NORM_NV(NORM_BWD_ROW, T, R, VV, nv, s)
    NORM_TYPES(NORM_BWD);
  } else {
    const int tiles = (int)ceil_div64(D, 256);
    parts = ceil_div64(rows, NORM_DW_ROWS);
    DVAE_REQUIRE(launch_fits(parts * tiles, 256), "add_rms_norm_bwd: too large for one launch");
#define NORM_BWD_ANY(T, R, VV) \
  DVAE_LAUNCH((norm_bwd_any_kernel<T, R>), dim3((unsigned)q.rows), dim3(256), 0, s, q)
#define NORM_DW_ANY(T, R, VV) \
  DVAE_LAUNCH((norm_dw_any_kernel<T, R>), dim3((unsigned)(parts * tiles)), dim3(256), 0, s, p, tiles)
    const int e = dtype == DVAE_DT_F32 ? 4 : 2, re = rdtype == DVAE_DT_F32 ? 4 : 2;
    const int64_t span = norm_span(0);
    for (int64_t r0 = 0; r0 < rows; r0 += span) {
      const NormArgs q = norm_rows(p, r0, rows - r0 < span ? rows - r0 : span, e, re, e);
      NORM_TYPES(NORM_BWD_ANY);
    }
    NORM_TYPES(NORM_DW_ANY);
  }
  DVAE_LAUNCH(norm_dw_sum_kernel, dim3((unsigned)ceil_div64(D, 64)), dim3(64 * SUM_WAVES), 0, s, ws, dw, parts, (int)D);
  DVAE_LAUNCH_CHECK("add_rms_norm_bwd");
  return 0;
}
