// The global norm of many gradient tensors and their clipping by it.
//
//   norm = sqrt(sum over all tensors of g^2);  g -> g min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM: one read for the norm, one read and one write for the clipped values (no write, and
// no second read, where the tensors are clipped in place and nothing has to shrink). The squares are
// added in 64 bits: neither a gradient of 1e25 nor a billion small ones loses the norm.
// The tensors' table travels as the kernel's argument (no upload, nothing to keep alive, and a
// captured launch holds it), SLOTS tensors a launch, which keeps the arguments under 4 KB. A table's
// tensors are cut into tiles of TILE elements; block b takes tiles b, b + grid, ... and finds a tile's
// tensor by binary search over the first tiles (scalar loads of the argument). Partial sums go to one
// slot a block, and every block of the clipping launches adds all of them in the same order: no
// atomics, so equal gradients give equal bits, and no third launch between the two.
// Measured: 2.24 GB of reads and writes and the second read, 742 us; 368 tensors of 32.8 MB together 44 us in
// six launches, where the host's passes over them take 157.
#include "common.h"
#include <algorithm>
#include <new>
#include <vector>

namespace {

constexpr int BT = 256;
constexpr int SLOTS = 128;
constexpr int TILE = 8192;      // elements: 32 f32 a thread, 8 loads of 16 bytes in flight
constexpr int MAXGRID = 2048;   // 8 blocks a CU

struct Table {
  void* p[SLOTS];
  int64_t n[SLOTS];       // elements; negative: bf16
  int64_t at[SLOTS];      // first element in the flat output
  int32_t first[SLOTS];   // first tile
  int32_t count, tiles;
};

struct __attribute__((packed, aligned(4))) F4 { float e[4]; };
struct __attribute__((packed, aligned(2))) B8 { bf16_t e[8]; };

__device__ __forceinline__ int slot_of(const Table& t, int tile) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double v, double* sm) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = sm[0];
#pragma unroll
  for (int k = 1; k < BT / 64; ++k) s += sm[k];
  return s;
}

__global__ __launch_bounds__(BT) void grad_sq_kernel(const Table t, double* __restrict__ part) {
  __shared__ double sm[BT / 64];
  double s = 0.0;
  for (int tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const int k = slot_of(t, tile);
    const int64_t cnt = t.n[k], n = cnt < 0 ? -cnt : cnt;
    const int64_t a = (int64_t)(tile - t.first[k]) * TILE;
    const int m = (int)min((int64_t)TILE, n - a);
    if (cnt < 0) {
      const bf16_t* g = (const bf16_t*)t.p[k] + a;
#pragma unroll 4
      for (int i = threadIdx.x * 8; i + 8 <= m; i += BT * 8) {
        const B8 v = *reinterpret_cast<const B8*>(g + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fma((double)(float)v.e[e], (double)(float)v.e[e], s);
      }
      const int i = (m & ~7) + threadIdx.x;
      if (i < m) s = fma((double)(float)g[i], (double)(float)g[i], s);
    } else {
      const float* g = (const float*)t.p[k] + a;
#pragma unroll 8
      for (int i = threadIdx.x * 4; i + 4 <= m; i += BT * 4) {
        const F4 v = *reinterpret_cast<const F4*>(g + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fma((double)v.e[e], (double)v.e[e], s);
      }
      const int i = (m & ~3) + threadIdx.x;
      if (i < m) s = fma((double)g[i], (double)g[i], s);
    }
  }
  s = block_sum(s, sm);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <typename TI, typename TO>
__device__ __forceinline__ void scale_tile(const TI* src, TO* dst, int m, float coef) {
  // 4 elements a thread and step: 16-byte loads and stores of f32, 8-byte ones of bf16
  struct __attribute__((packed, aligned(sizeof(TI)))) In { TI e[4]; };
  struct __attribute__((packed, aligned(sizeof(TO)))) Out { TO e[4]; };
#pragma unroll 8
  for (int i = threadIdx.x * 4; i + 4 <= m; i += BT * 4) {
    const In v = *reinterpret_cast<const In*>(src + i);
    Out o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.e[e] = from_f32<TO>(to_f32(v.e[e]) * coef);
    *reinterpret_cast<Out*>(dst + i) = o;
  }
  const int i = (m & ~3) + threadIdx.x;
  if (i < m) dst[i] = from_f32<TO>(to_f32(src[i]) * coef);
}

__global__ __launch_bounds__(BT) void grad_scale_kernel(const Table t, const double* __restrict__ part, int parts,
                                                        float max_norm, float* __restrict__ norm, void* out,
                                                        int out_bf16) {
  __shared__ double sm[BT / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += BT) s += part[i];
  s = block_sum(s, sm);
  const double len = sqrt(s);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)len;
  // NaN stays (it fails the comparison): the clipped gradients then show it
  const double c = (double)max_norm / (len + 1e-6);
  const float coef = c > 1.0 ? 1.f : (float)c;
  if (!out && coef == 1.f) return;
  // backwards: what the norm's pass read last is still in the 256 MB behind the L2
  for (int tile = t.tiles - 1 - blockIdx.x; tile >= 0; tile -= gridDim.x) {
    const int k = slot_of(t, tile);
    const int64_t cnt = t.n[k], n = cnt < 0 ? -cnt : cnt;
    const int64_t a = (int64_t)(tile - t.first[k]) * TILE;
    const int m = (int)min((int64_t)TILE, n - a);
    const int64_t o = t.at[k] + a;
    if (cnt < 0) {
      bf16_t* g = (bf16_t*)t.p[k] + a;
      if (!out) scale_tile<bf16_t, bf16_t>(g, g, m, coef);
      else if (out_bf16) scale_tile<bf16_t, bf16_t>(g, (bf16_t*)out + o, m, coef);
      else scale_tile<bf16_t, float>(g, (float*)out + o, m, coef);
    } else {
      float* g = (float*)t.p[k] + a;
      if (!out) scale_tile<float, float>(g, g, m, coef);
      else if (out_bf16) scale_tile<float, bf16_t>(g, (bf16_t*)out + o, m, coef);
      else scale_tile<float, float>(g, (float*)out + o, m, coef);
    }
  }
}

// no two of the tensors (nor one of them and the output) share a byte: a shared one would be scaled
// twice, or by two blocks at once
static int disjoint(void* const* ptr, const int64_t* n, const int32_t* dt, int count, const void* out, int64_t bytes) {
  try {
    std::vector<std::pair<uintptr_t, uintptr_t>> r;
    r.reserve(count + 1);
    for (int i = 0; i < count; ++i)
      if (n[i]) r.emplace_back((uintptr_t)ptr[i], (uintptr_t)ptr[i] + n[i] * (dt[i] == DP_BF16 ? 2 : 4));
    if (out && bytes) r.emplace_back((uintptr_t)out, (uintptr_t)out + bytes);
    std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i)
      DP_REQUIRE(r[i].first >= r[i - 1].second, "dp_grad_clip: two of the tensors share memory");
  } catch (const std::bad_alloc&) {
    dp_set_error("dp_grad_clip: out of host memory");
    return DP_EINVAL;
  }
  return 0;
}

}  // namespace

extern "C" int64_t dp_grad_clip_ws_bytes(int32_t count) {
  return count > 0 ? (int64_t)((count + SLOTS - 1) / SLOTS) * MAXGRID * 8 : 0;
}

extern "C" int dp_grad_clip(void* const* ptr, const int64_t* n, const int32_t* dtype, int32_t count, float max_norm,
                            float* norm, void* out, int64_t out_n, int32_t out_dtype, void* ws, int64_t ws_bytes,
                            void* stream) {
  DP_REQUIRE(ptr && n && dtype && norm && ws && count > 0, "dp_grad_clip: bad arguments");
  DP_REQUIRE(max_norm >= 0.f, "dp_grad_clip: max_norm %g", (double)max_norm);
  DP_REQUIRE(!out || out_dtype == DP_F32 || out_dtype == DP_BF16, "dp_grad_clip: output dtype %d", out_dtype);
  DP_REQUIRE(ws_bytes >= dp_grad_clip_ws_bytes(count), "dp_grad_clip: workspace holds %lld bytes, needs %lld",
             (long long)ws_bytes, (long long)dp_grad_clip_ws_bytes(count));
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    DP_REQUIRE(dtype[i] == DP_F32 || dtype[i] == DP_BF16, "dp_grad_clip: tensor %d has dtype %d", i, dtype[i]);
    DP_REQUIRE(n[i] >= 0 && (ptr[i] || !n[i]), "dp_grad_clip: tensor %d: %lld elements at %p", i, (long long)n[i],
               ptr[i]);
    total += n[i];
  }
  DP_REQUIRE(total / TILE + count < INT32_MAX, "dp_grad_clip: %lld elements are too many", (long long)total);
  DP_REQUIRE(!out || out_n == total, "dp_grad_clip: the output holds %lld elements, the tensors %lld",
             (long long)out_n, (long long)total);
  if (const int rc = disjoint(ptr, n, dtype, count, out, out ? out_n * (out_dtype == DP_BF16 ? 2 : 4) : 0)) return rc;
  hipStream_t s = as_stream(stream);
  double* part = (double*)ws;
  const int tables = (count + SLOTS - 1) / SLOTS;
  auto fill = [&](int base, int64_t at) {
    Table t;
    t.count = std::min(SLOTS, count - base);
    t.tiles = 0;
    for (int i = 0; i < t.count; ++i) {
      const int64_t m = n[base + i];
      t.p[i] = ptr[base + i];
      t.n[i] = dtype[base + i] == DP_BF16 ? -m : m;
      t.at[i] = at;
      t.first[i] = t.tiles;   // a tensor of no elements has no tile: the search passes over it
      t.tiles += (int)((m + TILE - 1) / TILE);
      at += m;
    }
    return t;
  };
  int parts = 0;
  for (int k = 0; k < tables; ++k) {
    const Table t = fill(k * SLOTS, 0);
    const int grid = std::min(t.tiles, MAXGRID);
    if (!grid) continue;
    hipLaunchKernelGGL(grad_sq_kernel, dim3(grid), dim3(BT), 0, s, t, part + parts);
    parts += grid;
  }
  int64_t at = total;
  for (int k = tables - 1; k >= 0; --k) {
    for (int i = k * SLOTS; i < std::min(count, (k + 1) * SLOTS); ++i) at -= n[i];
    const Table t = fill(k * SLOTS, at);
    const int grid = std::min(t.tiles, MAXGRID);
    if (grid || k == 0)
      hipLaunchKernelGGL(grad_scale_kernel, dim3(std::max(1, grid)), dim3(BT), 0, s, t, part, parts, max_norm,
                         k ? nullptr : norm, out, out_dtype == DP_BF16);
  }
  return dp_check_launch("dp_grad_clip");
}
