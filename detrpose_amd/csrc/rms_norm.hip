// Root-mean-square norm with the residual's addition: forward, backward, and the e4m3 form.
//
//   r = x + res (rounded to the activations' type: what the residual stream holds, and what the
//   backward reads again), rstd = 1 / sqrt(mean r^2 + eps), y = r rstd w
//   dr = rstd (w dy - rh mean(w dy rh)) + dres with rh = r rstd, dw = sum over rows of dy rh
//
// Sums, rstd and dw are f32 throughout. Bound by HBM: the forward reads x, res and writes r, y once
// each, the backward reads r, dy, dres and writes dr; a row stays in registers between the passes.
// TPR threads own a row (up to 64: lanes of one wave, no barrier; from 256: one block), each V vectors of 16 bytes at
// vector index t + TPR i, so every access of a wave is 1 KB contiguous. Rows need only their
// element's alignment (the loads are declared so and stay 16 bytes wide); the last, partial vector
// of a row whose length is no multiple of the vector is read and written element by element.
// Measured (the least of 25 launches), 8192 x 4096 bf16 with residual: forward 47 us and backward 47 + 6 (the sum over dw's parts) of 268 MB
// each, 5.7 and 5.0 TB/s (what lies in the 256 MB behind the L2 is read faster than HBM); the e4m3 form 8.5 us
// of 18.5 MB.
#include "common.h"
#include <algorithm>

namespace {

constexpr int BT = 256;         // threads of a block whose rows take no more
constexpr int MOST = 2 * 1024;  // vectors of a row at most
template <int TPR> constexpr int threads() { return TPR > BT ? TPR : BT; }

template <typename T> constexpr int vn() { return 16 / (int)sizeof(T); }

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Raw16 {
  T e[16 / sizeof(T)];
};

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// vector i of a row of c elements, as it lies there (zero past the end), and its elements as f32
template <typename T>
__device__ __forceinline__ u32x4_t raw_load(const T* __restrict__ p, int i, int c) {
  constexpr int N = vn<T>();
  const int at = i * N;
  if (at + N <= c) return __builtin_bit_cast(u32x4_t, *reinterpret_cast<const Raw16<T>*>(p + at));
  u32x4_t u = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if (at + e >= c) continue;
    if constexpr (sizeof(T) == 2) u[e / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[at + e]) << (16 * (e & 1));
    else u[e] = __builtin_bit_cast(uint32_t, p[at + e]);
  }
  return u;
}
template <typename T>
__device__ __forceinline__ float element(const u32x4_t& u, int e) {
  if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
  else return __uint_as_float(u[e]);
}
template <typename T>
__device__ __forceinline__ void row_load(const T* __restrict__ p, int i, int c, float (&v)[vn<T>()]) {
  const u32x4_t u = raw_load<T>(p, i, c);
#pragma unroll
  for (int e = 0; e < vn<T>(); ++e) v[e] = element<T>(u, e);
}

template <typename T, int N>
__device__ __forceinline__ void row_store(T* __restrict__ p, int i, int c, const float (&v)[N]) {
  constexpr int VN = vn<T>();
  static_assert(N % VN == 0, "whole vectors");
#pragma unroll
  for (int k = 0; k < N / VN; ++k) {
    const int at = i * N + k * VN;
    if (at + VN <= c) {
      Raw16<T> u;
#pragma unroll
      for (int e = 0; e < VN; ++e) u.e[e] = from_f32<T>(v[k * VN + e]);
      *reinterpret_cast<Raw16<T>*>(p + at) = u;
    } else {
#pragma unroll
      for (int e = 0; e < VN; ++e)
        if (at + e < c) p[at + e] = from_f32<T>(v[k * VN + e]);
    }
  }
}

// the weights of vector i: f32 or the activations' type
template <typename T, typename W>
__device__ __forceinline__ void weight_load(const W* __restrict__ w, int i, int c, float (&v)[vn<T>()]) {
  constexpr int N = vn<T>(), M = vn<W>();
  constexpr int P = N < M ? N : M;
  const int at = i * N;
#pragma unroll
  for (int k = 0; k < N; k += P) {
    if (at + k + P <= c) {
      struct __attribute__((packed, aligned(sizeof(W)))) Part { W e[P]; };
      const Part u = *reinterpret_cast<const Part*>(w + at + k);
#pragma unroll
      for (int e = 0; e < P; ++e) v[k + e] = to_f32(u.e[e]);
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) v[k + e] = at + k + e < c ? to_f32(w[at + k + e]) : 0.f;
    }
  }
}

// sum (or maximum) over the TPR threads of a row; red: one slot per wave, one call's own
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
    const float u = __shfl_xor(v, o, 64);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int k = 1; k < TPR / 64; ++k) s = MAX ? fmaxf(s, red[k]) : s + red[k];
    v = s;
  }
  return v;
}

// four values to e4m3 (round to nearest even, NaN kept), one dword
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (unsigned)w;
}

template <typename T, typename W, int TPR, int V, bool E4M3>
__global__ __launch_bounds__(threads<TPR>()) void rms_fwd_kernel(void* __restrict__ yv, float* __restrict__ scale,
                                                     T* __restrict__ r, float* __restrict__ rstd_out,
                                                     const T* __restrict__ x, int64_t ld_x,
                                                     const T* __restrict__ res, int64_t ld_res,
                                                     const W* __restrict__ w, float eps, int rows, int c) {
  constexpr int N = vn<T>();
  __shared__ float red[2][threads<TPR>() / 64];
  const int row = blockIdx.x * (threads<TPR>() / TPR) + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  if (row >= rows) return;   // TPR >= 256: one row a block, uniform; else no barrier below
  const T* xp = x + (int64_t)row * ld_x;
  const T* rp = res ? res + (int64_t)row * ld_res : nullptr;
  T* sp = r ? r + (int64_t)row * c : nullptr;
  float a[V][N];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) row_load<T>(xp, t + TPR * i, c, a[i]);
  if (rp) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float b[N];
      row_load<T>(rp, t + TPR * i, c, b);
#pragma unroll
      for (int e = 0; e < N; ++e) a[i][e] = to_f32(from_f32<T>(a[i][e] + b[e]));
      if (sp) row_store<T, N>(sp, t + TPR * i, c, a[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) ss = fmaf(a[i][e], a[i][e], ss);
  ss = row_reduce<TPR, false>(ss, red[0]);
  const float rstd = 1.f / sqrtf(ss / (float)c + eps);
  if (rstd_out && t == 0) rstd_out[row] = rstd;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float wv[N];
    weight_load<T, W>(w, t + TPR * i, c, wv);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      a[i][e] = a[i][e] * rstd * wv[e];
      if (E4M3) top = fmaxf(top, fabsf(a[i][e]));
    }
    if (!E4M3) row_store<T, N>((T*)yv + (int64_t)row * c, t + TPR * i, c, a[i]);
  }
  if constexpr (E4M3) {
    // scale = max |y| / 448; a row of zeros gets scale 0 and zeros (its values stand for 0 x 0). Below the
    // normal numbers the quotient rounds so far that max |y| / scale passes 448, which e4m3 has no number for
    top = row_reduce<TPR, true>(top, red[1]);
    const float sc = top > 0.f ? fmaxf(top / 448.f, 0x1p-126f) : 0.f;
    if (t == 0) scale[row] = sc;
    uint8_t* yp = (uint8_t*)yv + (int64_t)row * c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = (t + TPR * i) * N;
      uint32_t q[N / 4];
#pragma unroll
      for (int e = 0; e < N; ++e) a[i][e] = sc > 0.f ? a[i][e] / sc : a[i][e] * 0.f;
#pragma unroll
      for (int k = 0; k < N / 4; ++k) q[k] = pack_e4m3(a[i][4 * k], a[i][4 * k + 1], a[i][4 * k + 2], a[i][4 * k + 3]);
      if (at + N <= c) {
        struct __attribute__((packed, aligned(1))) Out { uint32_t d[N / 4]; };
        Out o;
#pragma unroll
        for (int k = 0; k < N / 4; ++k) o.d[k] = q[k];
        *reinterpret_cast<Out*>(yp + at) = o;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (at + e < c) yp[at + e] = (uint8_t)(q[e / 4] >> (8 * (e % 4)));
      }
    }
  }
}

// A block walks rows blockIdx, + grid, ... (as many at once as it holds), the next row's loads in flight
// while this one is reduced; its dw stays in registers, is added over the block's rows at once, and is written
// once, part[block][c]; rms_dw_kernel adds the parts in a fixed order.
template <typename T, typename W, int TPR, int V>
__global__ __launch_bounds__(threads<TPR>()) void rms_bwd_kernel(T* __restrict__ dx, float* __restrict__ part,
                                                     const T* __restrict__ r, int64_t ld_r,
                                                     const float* __restrict__ rstd, const T* __restrict__ dy,
                                                     int64_t ld_dy, const T* __restrict__ dres, int64_t ld_dres,
                                                     const W* __restrict__ w, int rows, int c) {
  constexpr int N = vn<T>(), RPB = threads<TPR>() / TPR;
  __shared__ float red[2][threads<TPR>() / 64];
  __shared__ float dws[RPB > 1 ? BT * V * N : 1];
  const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int64_t step = (int64_t)gridDim.x * RPB;
  float dw[V][N], wv[V][N];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    weight_load<T, W>(w, t + TPR * i, c, wv[i]);
#pragma unroll
    for (int e = 0; e < N; ++e) dw[i][e] = 0.f;
  }
  u32x4_t rr[V], rg[V], rd[V];
  float rs = 0.f;
  auto fetch = [&](int64_t row) __attribute__((always_inline)) {
    if (row >= rows) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      rr[i] = raw_load<T>(r + row * ld_r, t + TPR * i, c);
      rg[i] = raw_load<T>(dy + row * ld_dy, t + TPR * i, c);
      if (dres) rd[i] = raw_load<T>(dres + row * ld_dres, t + TPR * i, c);
    }
    rs = rstd[row];
  };
  int64_t row = (int64_t)blockIdx.x * RPB + sub;
  fetch(row);
  int flip = 0;
  for (; row < rows; row += step) {
    float a[V][N], g[V][N];
    u32x4_t b[V];
    const float s = rs;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      b[i] = rd[i];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a[i][e] = element<T>(rr[i], e) * s;
        g[i][e] = element<T>(rg[i], e);
      }
    }
    fetch(row + step);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        dw[i][e] = fmaf(g[i][e], a[i][e], dw[i][e]);
        g[i][e] *= wv[i][e];
        dot = fmaf(g[i][e], a[i][e], dot);
      }
    }
    dot = row_reduce<TPR, false>(dot, red[flip]) / (float)c;
    flip ^= 1;   // the other slots next: a wave may still read these
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = s * (g[i][e] - a[i][e] * dot);
        g[i][e] = dres ? d + element<T>(b[i], e) : d;
      }
      row_store<T, N>(dx + row * c, t + TPR * i, c, g[i]);
    }
  }
  float* out = part + (int64_t)blockIdx.x * c;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) row_store<float, N>(out, t + TPR * i, c, dw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) dws[sub * (TPR * V * N) + (t + TPR * i) * N + e] = dw[i][e];
    __syncthreads();
    for (int j = threadIdx.x; j < c; j += BT) {
      float x = dws[j];
#pragma unroll
      for (int k = 1; k < RPB; ++k) x += dws[k * (TPR * V * N) + j];
      out[j] = x;
    }
  }
}

// dw[j] = sum over parts, in order: 16 columns x 16 groups of parts a block
template <typename W>
__global__ __launch_bounds__(BT) void rms_dw_kernel(W* __restrict__ dw, const float* __restrict__ part, int parts,
                                                    int c) {
  __shared__ float sm[BT];
  const int col = threadIdx.x & 15, j = blockIdx.x * 16 + col, grp = threadIdx.x >> 4;
  float s = 0.f;
  if (j < c) {
    const int n = (parts + 15) / 16, p0 = grp * n, p1 = min(parts, p0 + n);
#pragma unroll 8
    for (int p = p0; p < p1; ++p) s += part[(int64_t)p * c + j];
  }
  sm[threadIdx.x] = s;
  __syncthreads();
  if (grp == 0 && j < c) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += sm[16 * k + col];
    dw[j] = from_f32<W>(s);
  }
}

// Threads a row and vectors a thread (two at most: the backward keeps a row, the next one, the weights and dw) for
// rows of c elements: as few lanes as hold a row of up to 64 vectors, a wave for up to 128, else a block
struct Shape { int tpr, v; };
static Shape shape_of(int c, int n) {
  const int vec = (c + n - 1) / n;
  Shape s{8, 1};
  while (s.tpr < vec && s.tpr < 64) s.tpr *= 2;
  if (vec > 128) s.tpr = vec > 1024 ? 1024 : vec > 512 ? 512 : 256;
  if (s.tpr < vec) s.v = 2;
  if (s.tpr > 256) s.v = 2;
  return s;
}

// blocks of the backward: up to 4 a CU
static int bwd_parts(int rows, const Shape& s) {
  const int rpb = std::max(1, BT / s.tpr);
  return std::min(1024, (rows + rpb - 1) / rpb);
}

struct FwdArgs {
  void* y; float* scale; void* r; float* rstd; const void* x; int64_t ld_x; const void* res; int64_t ld_res;
  const void* w; float eps; int rows, c; hipStream_t s;
};

template <typename T, typename W, int TPR, int V, bool E4M3>
void fwd_launch(const FwdArgs& a) {
  constexpr int rpb = threads<TPR>() / TPR;
  constexpr int most = (int)(UINT32_MAX / threads<TPR>()) * rpb;   // rows of a launch: a grid has less than 2^32 threads
  for (int64_t r0 = 0; r0 < a.rows; r0 += most) {
    const int rows = (int)std::min<int64_t>(most, a.rows - r0);
    hipLaunchKernelGGL((rms_fwd_kernel<T, W, TPR, V, E4M3>), dim3((rows + rpb - 1) / rpb), dim3(threads<TPR>()), 0, a.s,
                       (char*)a.y + r0 * a.c * (E4M3 ? 1 : sizeof(T)), a.scale ? a.scale + r0 : nullptr,
                       a.r ? (T*)a.r + r0 * a.c : nullptr, a.rstd ? a.rstd + r0 : nullptr, (const T*)a.x + r0 * a.ld_x,
                       a.ld_x, a.res ? (const T*)a.res + r0 * a.ld_res : nullptr, a.ld_res, (const W*)a.w, a.eps, rows,
                       a.c);
  }
}

template <typename T, typename W, bool E4M3>
int fwd_shape(const FwdArgs& a) {
  const Shape s = shape_of(a.c, vn<T>());
#define DP_RMS_CASE(TPR_, V_) \
  if (s.tpr == TPR_ && s.v == V_) { fwd_launch<T, W, TPR_, V_, E4M3>(a); return dp_check_launch("dp_rms_norm"); }
  DP_RMS_CASE(8, 1) DP_RMS_CASE(16, 1) DP_RMS_CASE(32, 1)
  DP_RMS_CASE(64, 1) DP_RMS_CASE(64, 2) DP_RMS_CASE(256, 1)
  DP_RMS_CASE(256, 2) DP_RMS_CASE(512, 2) DP_RMS_CASE(1024, 2)
#undef DP_RMS_CASE
  dp_set_error("dp_rms_norm: rows of %d elements are too long", a.c);
  return DP_EINVAL;
}

template <bool E4M3>
int fwd_types(const FwdArgs& a, int dtype, int w_dtype) {
  if (dtype == DP_F32) return fwd_shape<float, float, E4M3>(a);
  return w_dtype == DP_F32 ? fwd_shape<bf16_t, float, E4M3>(a) : fwd_shape<bf16_t, bf16_t, E4M3>(a);
}

static int check_types(int dtype, int w_dtype, int c) {
  DP_REQUIRE(dtype == DP_F32 || dtype == DP_BF16, "dp_rms_norm: dtype %d", dtype);
  DP_REQUIRE(w_dtype == DP_F32 || w_dtype == dtype, "dp_rms_norm: weights are f32 or of the activations' type");
  const int most = MOST * (dtype == DP_F32 ? 4 : 8);
  DP_REQUIRE(c > 0 && c <= most, "dp_rms_norm: rows of %d elements (1 to %d)", c, most);
  return 0;
}

template <typename T, typename W>
int bwd_shape(void* dx, float* part, const void* r, int64_t ld_r, const float* rstd, const void* dy, int64_t ld_dy,
              const void* dres, int64_t ld_dres, const void* w, void* dw, int rows, int c, hipStream_t st) {
  const Shape s = shape_of(c, vn<T>());
  const int parts = bwd_parts(rows, s);
#define DP_RMS_CASE(TPR_, V_)                                                                                        \
  if (s.tpr == TPR_ && s.v == V_)                                                                                    \
    hipLaunchKernelGGL((rms_bwd_kernel<T, W, TPR_, V_>), dim3(parts), dim3(threads<TPR_>()), 0, st, (T*)dx, part, (const T*)r, ld_r, \
                       rstd, (const T*)dy, ld_dy, (const T*)dres, ld_dres, (const W*)w, rows, c);
  DP_RMS_CASE(8, 1) DP_RMS_CASE(16, 1) DP_RMS_CASE(32, 1)
  DP_RMS_CASE(64, 1) DP_RMS_CASE(64, 2) DP_RMS_CASE(256, 1)
  DP_RMS_CASE(256, 2) DP_RMS_CASE(512, 2) DP_RMS_CASE(1024, 2)
#undef DP_RMS_CASE
  hipLaunchKernelGGL((rms_dw_kernel<W>), dim3((c + 15) / 16), dim3(BT), 0, st, (W*)dw, part, parts, c);
  return dp_check_launch("dp_rms_norm_bwd");
}

}  // namespace

extern "C" int dp_rms_norm(void* y, void* r, float* rstd, const void* x, int64_t ld_x, const void* res,
                           int64_t ld_res, const void* weight, int32_t w_dtype, float eps, int32_t rows, int32_t c,
                           int32_t dtype, void* stream) {
  DP_REQUIRE(y && x && weight && rows >= 0, "dp_rms_norm: bad arguments");
  DP_REQUIRE(!r || res, "dp_rms_norm: r is written only with a residual");
  if (const int rc = check_types(dtype, w_dtype, c)) return rc;
  if (rows == 0) return 0;
  return fwd_types<false>({y, nullptr, r, rstd, x, ld_x, res, ld_res, weight, eps, rows, c, as_stream(stream)}, dtype,
                          w_dtype);
}

extern "C" int dp_rms_norm_e4m3(void* y, float* scale, void* r, const void* x, int64_t ld_x, const void* res,
                                int64_t ld_res, const void* weight, int32_t w_dtype, float eps, int32_t rows,
                                int32_t c, int32_t dtype, void* stream) {
  DP_REQUIRE(y && scale && x && weight && rows >= 0, "dp_rms_norm_e4m3: bad arguments");
  DP_REQUIRE(!r || res, "dp_rms_norm_e4m3: r is written only with a residual");
  if (const int rc = check_types(dtype, w_dtype, c)) return rc;
  if (rows == 0) return 0;
  return fwd_types<true>({y, scale, r, nullptr, x, ld_x, res, ld_res, weight, eps, rows, c, as_stream(stream)}, dtype,
                         w_dtype);
}

extern "C" int64_t dp_rms_norm_bwd_ws_floats(int32_t rows, int32_t c, int32_t dtype) {
  if (rows <= 0 || c <= 0 || c > MOST * (dtype == DP_F32 ? 4 : 8)) return 0;
  return (int64_t)bwd_parts(rows, shape_of(c, dtype == DP_F32 ? 4 : 8)) * c;
}

extern "C" int dp_rms_norm_bwd(void* dx, void* dweight, const void* r, int64_t ld_r, const float* rstd,
                               const void* dy, int64_t ld_dy, const void* dres, int64_t ld_dres, const void* weight,
                               int32_t w_dtype, float* ws, int64_t ws_floats, int32_t rows, int32_t c, int32_t dtype,
                               void* stream) {
  DP_REQUIRE(dx && dweight && r && rstd && dy && weight && ws && rows > 0, "dp_rms_norm_bwd: bad arguments");
  if (const int rc = check_types(dtype, w_dtype, c)) return rc;
  DP_REQUIRE(ws_floats >= dp_rms_norm_bwd_ws_floats(rows, c, dtype),
             "dp_rms_norm_bwd: workspace holds %lld floats, needs dp_rms_norm_bwd_ws_floats = %lld",
             (long long)ws_floats, (long long)dp_rms_norm_bwd_ws_floats(rows, c, dtype));
  hipStream_t s = as_stream(stream);
  if (dtype == DP_F32)
    return bwd_shape<float, float>(dx, ws, r, ld_r, rstd, dy, ld_dy, dres, ld_dres, weight, dweight, rows, c, s);
  if (w_dtype == DP_F32)
    return bwd_shape<bf16_t, float>(dx, ws, r, ld_r, rstd, dy, ld_dy, dres, ld_dres, weight, dweight, rows, c, s);
  return bwd_shape<bf16_t, bf16_t>(dx, ws, r, ld_r, rstd, dy, ld_dy, dres, ld_dres, weight, dweight, rows, c, s);
}
