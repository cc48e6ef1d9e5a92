// Attention over packed sequences, backward (packed_attn.h has the layouts).
//
//   p = exp(s - lse), dp = dO V^T, D = sum_d dO O, ds = p (dp - D)
//   dQ = scale ds K, dK = scale ds^T Q, dV = p^T dO, dbias[bucket][head] = sum of ds in the bucket
//
// Two kernels, each owner of what it writes, so nothing is added atomically and equal inputs give
// equal bits: packed_bwd_q_kernel walks the keys of a tile of 128 rows (S^T, dP^T, dQ^T: three products)
// and stores D; packed_bwd_kv_kernel walks the rows (all heads of the group, so grouped heads are summed
// in the accumulators) of a tile of 128 keys (S, dP, dV^T, dK^T: four products). Two of the seven products
// are done twice in exchange. p and ds are rounded to bf16 for their products, as p in the forward.
//
// The table's gradient comes from the first kernel: each lane owns one row (one head), so it adds its
// ds into its own LDS bins [bucket][thread] (a 4-byte add with no other lane at that address; one add
// per tile where the whole tile lies in one bucket); the block then adds the bins of a head's rows and
// writes one part per block, and packed_dbias_kernel adds the parts, all in fixed orders.
#include "packed_attn.h"
#include <algorithm>

int dp_packed_attn_args(const dp_packed_attn* d, dppa::Args* a, const char* what, bool backward);

namespace {
using namespace dppa;

// WK waves of a block share its rows and take the key tile's subtiles in turn, as in the forward
template <typename T, int DP, int WK, int BN, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 4 && DP == 128 ? 1 : 2) void packed_bwd_q_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int TB = TL::bytes(BN), NS = BN / 32 / WK, ROWS = BM / WK, OP = DP + 4;
  static_assert(WK == 1 || 4 * TB >= 4 * 32 * OP * 4, "the join of the waves fits the tiles");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform: scalar branches below
  const int wk = wave % WK, wr = wave / WK;
  const int kvh = uniform(blockIdx.x % a.hkv), tile = a.tiles - 1 - blockIdx.x / a.hkv;
  const int heads = a.hkv * a.group;
  float* part = BIAS ? a.dbias_part + ((int64_t)tile * a.hkv + kvh) * a.group * a.buckets : nullptr;
  Item it;
  if (!find_item(a.cu_q, a.tq, a.cu_k, a.tk, a.nseq, true, tile,
                 [&](int len, int) { return (len * a.group + ROWS - 1) / ROWS; }, it)) {
    if constexpr (BIAS)
      for (int i = threadIdx.x; i < a.group * a.buckets; i += NT) part[i] = 0.f;
    return;
  }
  const int q0 = it.start, lq = it.len, k0 = it.start2, lk = it.len2;
  const int off = lk - lq, rows = lq * a.group, row0 = it.sub * ROWS;
  const int first = row0 + 32 * wr, r = first + (lane & 31);
  const bool ok = r < rows;
  const int rc = min(r, rows - 1), pos = rc / a.group, g = rc - pos * a.group, head = kvh * a.group + g;
  auto limit = [&](int row) {
    return a.causal ? clampi(min(row, rows - 1) / a.group + off + 1, 0, lk) : lk;
  };
  const int lim = limit(r), wmin = uniform(limit(first)), wmax = uniform(first < rows ? limit(first + 31) : 0);
  const int nt = uniform((limit(row0 + ROWS - 1) + BN - 1) / BN);
  // positions of the wave's first and last row
  const int pfirst = uniform(first / a.group + off), plast = uniform(min(first + 31, rows - 1) / a.group + off);
  Bias bias{};
  float* bins = nullptr;
  if constexpr (BIAS) {
    bins = reinterpret_cast<float*>(smem + 4 * TB);
    for (int b = 0; b < a.buckets; ++b) bins[b * NT + threadIdx.x] = 0.f;   // the thread's own
    bias = bias_setup<T>(a, smem + 4 * TB + a.buckets * NT * 4, kvh);
    bins += threadIdx.x;
  }

  const int64_t at = (int64_t)(q0 + pos) * heads + head;
  u32x4 qf[TL::KS], gf[TL::KS];
  load_frags<T, DP>((const T*)a.q + (int64_t)(q0 + pos) * a.q_row + head * a.q_head, ok, a.dim, h, qf);
  load_frags<T, DP>((const T*)a.dout + (int64_t)(q0 + pos) * a.g_row + head * a.g_head, ok, a.dim, h, gf);
  float D = 0.f;
  {
    u32x4 of[TL::KS];
    load_frags<T, DP>((const T*)a.out + (int64_t)(q0 + pos) * a.o_row + head * a.o_head, ok, a.dim, h, of);
#pragma unroll
    for (int s = 0; s < TL::KS; ++s) {
      const T* x = reinterpret_cast<const T*>(&of[s]);
      const T* y = reinterpret_cast<const T*>(&gf[s]);
#pragma unroll
      for (int e = 0; e < TL::VN; ++e) D = fmaf(to_f32(x[e]), to_f32(y[e]), D);
    }
    D = half_sum(D);
  }
  if (ok && h == 0 && wk == 0) a.dsum[at] = D;
  const float lse = ok ? a.lse[at] : INFINITY;

  const int ks = (int)(a.k_row * sizeof(T)), vs = (int)(a.v_row * sizeof(T));
  const int koff = lane_off<T, DP>(ks, a.dim), voff = lane_off<T, DP>(vs, a.dim);
  auto fetch = [&](int j) {
    char* buf = smem + (j & 1) * 2 * TB;
    const int key0 = j * BN, left = lk - key0;
    stage_rows<T, DP, BN>((const T*)a.k + (int64_t)(k0 + key0) * a.k_row + kvh * a.k_head, ks, left, buf, a.dim, koff,
                          wave);
    stage_rows<T, DP, BN>((const T*)a.v + (int64_t)(k0 + key0) * a.v_row + kvh * a.v_head, vs, left, buf + TB, a.dim,
                          voff, wave);
  };

  const float c = a.scale * LOG2E;
  f32x16 dq[TL::ND];
#pragma unroll
  for (int t = 0; t < TL::ND; ++t) dq[t] = zero16();

  dpconv::wait_vmcnt<0>();   // the row loads above, so that the loop's waits count tiles only
  if (nt > 0) fetch(0);
  for (int j = 0; j < nt; ++j) {
    tile_barrier();
    if (j + 1 < nt) fetch(j + 1);
    const char* buf = smem + (j & 1) * 2 * TB;
    const int key0 = j * BN;
    if (key0 >= wmax) continue;
#pragma unroll
    for (int un = 0; un < NS; ++un) {
      const int u = NS * wk + un, k32 = key0 + 32 * u;
      if (k32 >= wmax) break;
      f32x16 s = rows_mma<T, DP>(buf, u, lane, qf);
      const f32x16 dp = rows_mma<T, DP>(buf + TB, u, lane, gf);
      int one = -1;
      if constexpr (BIAS) {
        one = bias.one_bucket(k32 - plast, k32 + 31 - pfirst);
        const float* tab = bias.tab + g * bias.nb;
        if (one >= 0) {
          const float b = tab[one];
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], a.scale, b);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[i] = fmaf(s[i], a.scale, tab[bias.bucket(k32 + 8 * (i / 4) + 4 * h + (i & 3) - pos - off)]);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(BIAS ? (s[i] - lse) * LOG2E : fmaf(s[i], c, -lse));
        s[i] = p * (dp[i] - D);
      }
      if (k32 + 32 > wmin) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k32 + 8 * (i / 4) + 4 * h + (i & 3) >= lim) s[i] = 0.f;
      }
      if constexpr (BIAS) {
        if (one >= 0) {
          float t = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) t += s[i];
          bins[one * NT] += t;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            __hip_atomic_fetch_add(bins + bias.bucket(k32 + 8 * (i / 4) + 4 * h + (i & 3) - pos - off) * NT, s[i],
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
      cols_mma<T, DP>(buf, u, lane, s, dq);
    }
  }

  typedef T T4 __attribute__((ext_vector_type(4)));
  if constexpr (WK == 1) {
    if (ok) {
#pragma unroll
      for (int t = 0; t < TL::ND; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = 32 * t + 8 * e + 4 * h;
          if (d < a.dim) {
            T4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = from_f32<T>(dq[t][4 * e + i] * a.scale);
            *reinterpret_cast<T4*>((T*)a.dq + at * a.dim + d) = w;
          }
        }
    }
  } else {
    __syncthreads();
    float* oo = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int t = 0; t < TL::ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(oo + (wave * 32 + (lane & 31)) * OP + 32 * t + 8 * e + 4 * h) =
            f32x4{dq[t][4 * e], dq[t][4 * e + 1], dq[t][4 * e + 2], dq[t][4 * e + 3]};
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * (DP / 4); i += NT) {
      const int jr = i / (DP / 4), d = (i - jr * (DP / 4)) * 4, row = row0 + jr;
      if (row >= rows || d >= a.dim) continue;
      const int w0 = (jr >> 5) * WK * 32 + (jr & 31), rp = row / a.group;
      f32x4 sum = *reinterpret_cast<const f32x4*>(oo + w0 * OP + d);
#pragma unroll
      for (int w = 1; w < WK; ++w) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(oo + (w0 + 32 * w) * OP + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
      }
      T4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(sum[e] * a.scale);
      const int64_t x = (int64_t)(q0 + rp) * heads + kvh * a.group + row - rp * a.group;
      *reinterpret_cast<T4*>((T*)a.dq + x * a.dim + d) = w;
    }
  }
  if constexpr (BIAS) {
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(smem + 4 * TB);
    for (int p = threadIdx.x; p < a.group * a.buckets; p += NT) {
      const int pg = p / a.buckets, b = p - pg * a.buckets;
      int rr = (pg - row0 % a.group + a.group) % a.group;   // the block's first row of this head
      float t = 0.f;
      for (; rr < min(ROWS, rows - row0); rr += a.group)
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float* x = all + b * NT + ((rr >> 5) * WK + w) * 64 + (rr & 31);
          t += x[0] + x[32];
        }
      part[p] = t;
    }
  }
}

// dbias[bucket][head] = sum over tiles of the parts, in order: one block per head
template <typename TB>
__global__ __launch_bounds__(NT) void packed_dbias_kernel(TB* __restrict__ out, const float* __restrict__ part,
                                                          int tiles, int hkv, int group, int buckets) {
  __shared__ float sm[NT];
  const int head = blockIdx.x, kvh = head / group, g = head - kvh * group;
  const int b = threadIdx.x & 63, slice = threadIdx.x >> 6;
  float s = 0.f;
  if (b < buckets)
    for (int t = slice; t < tiles; t += NT / 64)
      s += part[(((int64_t)t * hkv + kvh) * group + g) * buckets + b];
  sm[threadIdx.x] = s;
  __syncthreads();
  if (slice == 0 && b < buckets)
    out[(int64_t)b * hkv * group + head] = from_f32<TB>((sm[b] + sm[64 + b]) + (sm[128 + b] + sm[192 + b]));
}

// rows [cut * step, ...) of a sequence's cuts
__device__ __forceinline__ int cuts_of(const Args& a, int rows) {
  return a.cuts <= 1 ? 1 : clampi((rows + a.cut_rows - 1) / a.cut_rows, 1, a.cuts);
}
__device__ __forceinline__ int cut_step(int rows, int cuts) { return ((rows + cuts - 1) / cuts + 31) / 32 * 32; }

template <typename T, int DP, int BR, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 2 ? 2 : 1) void packed_bwd_kv_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int TB = TL::bytes(BR), NS = BR / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  // per row of a tile: lse, D, and (for the bias) its position and head; two buffers, written a tile ahead
  float* lse_s = reinterpret_cast<float*>(smem + 4 * TB);
  float* dsum_s = lse_s + 2 * BR;
  int* pos_s = reinterpret_cast<int*>(dsum_s + 2 * BR);
  int* head_s = pos_s + 2 * BR;
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform: scalar branches below
  const int kvh = uniform(blockIdx.x % a.hkv);
  const int heads = a.hkv * a.group;
  auto tiles_of = [&](int len) { return (len + BM - 1) / BM; };
  Item it;
  if (!find_item(a.cu_k, a.tk, a.cu_q, a.tq, a.nseq, true, blockIdx.x / a.hkv,
                 [&](int len, int queries) { return tiles_of(len) * cuts_of(a, queries * a.group); }, it))
    return;
  const int k0 = it.start, lk = it.len, q0 = it.start2, lq = it.len2;
  const int off = lk - lq, rows = lq * a.group, ntile = tiles_of(lk);
  const int cuts = uniform(cuts_of(a, rows)), cut = uniform(it.sub / ntile), tile = it.sub - cut * ntile;
  const int first = tile * BM + 32 * wave, key = first + (lane & 31);
  const bool ok = key < lk;
  // the first row that sees a key
  auto sees = [&](int kk) { return a.causal ? max(0, kk - off) * a.group : 0; };
  const int mine = sees(key), wfirst = uniform(sees(first)), wlast = uniform(sees(min(first + 31, lk - 1)));
  // this block's rows [start, end)
  const int seen = sees(tile * BM) / 32 * 32, step = cuts > 1 ? cut_step(rows, cuts) : 0;
  const int start = uniform(max(seen, cut * step)), end = uniform(cuts > 1 ? min(rows, (cut + 1) * step) : rows);
  if (start >= end && cuts > 1) return;
  Bias bias{};
  if constexpr (BIAS) bias = bias_setup<T>(a, smem + 4 * TB + 16 * BR * 2, kvh);

  u32x4 kf[TL::KS], vf[TL::KS];
  load_frags<T, DP>((const T*)a.k + (int64_t)(k0 + min(key, lk - 1)) * a.k_row + kvh * a.k_head, ok, a.dim, h, kf);
  load_frags<T, DP>((const T*)a.v + (int64_t)(k0 + min(key, lk - 1)) * a.v_row + kvh * a.v_head, ok, a.dim, h, vf);

  const int nt = end > start ? (end - start + BR - 1) / BR : 0;
  const float invg = 1.f / (float)a.group;
  // lse and D of the next tile's rows are loaded with it and stored a step later
  float lse_r = INFINITY, dsum_r = 0.f;
  int pos_r = 0, head_r = 0;
  auto fetch = [&](int j) {
    char* buf = smem + (j & 1) * 2 * TB;
    const int r0 = start + j * BR, p0 = r0 / a.group, skip = r0 - p0 * a.group;
    const i32x4 rq = make_rsrc((const T*)a.q + (int64_t)(q0 + p0) * a.q_row + kvh * a.group * a.q_head);
    const i32x4 rg = make_rsrc((const T*)a.dout + (int64_t)(q0 + p0) * a.g_row + kvh * a.group * a.g_head);
    // (query, head) of the tile's row: a small quotient, exact in f32
    auto split = [&](int row, int& p, int& g) {
      p = (int)(((float)(skip + row) + 0.5f) * invg);
      g = skip + row - p * a.group;
    };
    auto at = [&](int row, int64_t rs, int64_t hs) {
      int p, g;
      split(row, p, g);
      return r0 + row < end ? p * (int)(rs * sizeof(T)) + g * (int)(hs * sizeof(T)) : -1;
    };
    stage<T, DP, BR>(rq, buf, a.dim, [&](int row) { return at(row, a.q_row, a.q_head); });
    stage<T, DP, BR>(rg, buf + TB, a.dim, [&](int row) { return at(row, a.g_row, a.g_head); });
    if (threadIdx.x < BR) {
      lse_r = INFINITY;   // a row past the end: p = 0
      dsum_r = 0.f;
      if (r0 + (int)threadIdx.x < end) {
        int p, g;
        split(threadIdx.x, p, g);
        const int64_t x = (int64_t)(q0 + p0 + p) * heads + kvh * a.group + g;
        lse_r = a.lse[x];
        dsum_r = a.dsum[x];
        pos_r = p0 + p;
        head_r = g;
      }
    }
  };
  auto publish = [&](int j) {
    if (threadIdx.x < BR) {
      const int x = (j & 1) * BR + threadIdx.x;
      lse_s[x] = lse_r;
      dsum_s[x] = dsum_r;
      if constexpr (BIAS) {
        pos_s[x] = pos_r;
        head_s[x] = head_r;
      }
    }
  };

  const float c = a.scale * LOG2E;
  f32x16 dk[TL::ND], dv[TL::ND];
#pragma unroll
  for (int t = 0; t < TL::ND; ++t) dk[t] = dv[t] = zero16();

  if (nt > 0) fetch(0);
  for (int j = 0; j < nt; ++j) {
    dpconv::wait_vmcnt<0>();
    publish(j);
    __syncthreads();
    if (j + 1 < nt) fetch(j + 1);
    const char* buf = smem + (j & 1) * 2 * TB;
    const int r0 = start + j * BR;
    if (first >= lk) continue;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const int r32 = r0 + 32 * u;
      if (r32 >= end) break;
      if (r32 + 31 < wfirst) continue;
      const int x0 = (j & 1) * BR + 32 * u + 4 * h;
      f32x16 s = rows_mma<T, DP>(buf, u, lane, kf);
      if constexpr (BIAS) {
        const int pf = r32 / a.group + off, pl = min(r32 + 31, rows - 1) / a.group + off;
        const int one = bias.one_bucket(first - pl, first + 31 - pf);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int x = x0 + 8 * (i / 4) + (i & 3);
          const int b = one >= 0 ? one : bias.bucket(key - pos_s[x] - off);
          s[i] = fmaf(s[i], a.scale, bias.tab[head_s[x] * bias.nb + b]);
        }
      }
      f32x16 p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(lse_s + x0 + 8 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = s[4 * e + i];
          p[4 * e + i] = __builtin_amdgcn_exp2f(BIAS ? (v - ls[i]) * LOG2E : fmaf(v, c, -ls[i]));
        }
      }
      if (r32 < wlast || !ok) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (r32 + 8 * (i / 4) + 4 * h + (i & 3) < mine || !ok) p[i] = 0.f;
      }
      cols_mma<T, DP>(buf + TB, u, lane, p, dv);
      const f32x16 dp = rows_mma<T, DP>(buf + TB, u, lane, vf);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x4 ds = *reinterpret_cast<const f32x4*>(dsum_s + x0 + 8 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[4 * e + i] *= dp[4 * e + i] - ds[i];
      }
      cols_mma<T, DP>(buf, u, lane, p, dk);
    }
  }

  if (ok) {
    const int64_t kr = (int64_t)(k0 + key) * a.hkv + kvh;
    float* part = a.kv_part + ((int64_t)cut * a.tk * a.hkv + kr) * 2 * a.dim;
#pragma unroll
    for (int t = 0; t < TL::ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * t + 8 * e + 4 * h;
        if (d < a.dim) {
          f32x4 x, y;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = dk[t][4 * e + i] * a.scale;
            y[i] = dv[t][4 * e + i];
          }
          if (cuts > 1) {
            *reinterpret_cast<f32x4*>(part + d) = x;
            *reinterpret_cast<f32x4*>(part + a.dim + d) = y;
          } else {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 u, w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              u[i] = from_f32<T>(x[i]);
              w[i] = from_f32<T>(y[i]);
            }
            *reinterpret_cast<T4*>((T*)a.dk + kr * a.dim + d) = u;
            *reinterpret_cast<T4*>((T*)a.dv + kr * a.dim + d) = w;
          }
        }
      }
    // the last cut's rows see every key: it says which cuts there are (and 0 of them where it wrote the result)
    if (a.cuts > 1 && cut == cuts - 1 && h == 0) a.kv_n[kr] = cuts > 1 ? (seen / step) << 16 | cuts : 0;
  }
}

// keys whose rows were cut: dk and dv = the sums of the parts in the order of the cuts, four elements a thread
template <typename T, int DP>
__global__ __launch_bounds__(NT) void packed_kv_join_kernel(const Args a) {
  constexpr int TPR = DP / 4;
  const int64_t all = (int64_t)a.tk * a.hkv;
  const int64_t kr = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const int d = (threadIdx.x % TPR) * 4;
  if (kr >= all || d >= a.dim) return;
  const int n = a.kv_n[kr], from = n >> 16, to = min(n & 0xffff, a.cuts);
  if (n <= 0) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
  for (int c = from; c < to; ++c) {
    const float* part = a.kv_part + (c * all + kr) * 2 * a.dim + d;
    const f32x4 u = *reinterpret_cast<const f32x4*>(part), w = *reinterpret_cast<const f32x4*>(part + a.dim);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] += u[i];
      y[i] += w[i];
    }
  }
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 u, w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u[i] = from_f32<T>(x[i]);
    w[i] = from_f32<T>(y[i]);
  }
  *reinterpret_cast<T4*>((T*)a.dk + kr * a.dim + d) = u;
  *reinterpret_cast<T4*>((T*)a.dv + kr * a.dim + d) = w;
}

// How the two kernels are cut. Lengths are on the device, so the rule goes by totals.
struct Plan { int wk, items, cut_rows, cuts, ktiles; };
static Plan plan_of(const dp_packed_attn* d) {
  const int64_t group = d->heads / d->kv_heads, rows = d->tq * group, seqs = std::max(1, d->nseq);
  Plan p{1, 0, 0, 1, 0};
  const int64_t wide = (rows / BM + 1) * d->kv_heads;
  if (wide < 256 && d->tk <= 2048 * seqs) p.wk = d->dtype == DP_F32 && d->dim > 64 ? 2 : 4;
  // the bins beside the waves' larger key tile: where both do not fit the LDS, the waves lie along the rows
  const int dp = d->dim <= 32 ? 32 : d->dim <= 64 ? 64 : 128, last = d->bias && d->buckets > 2 ? 4096 + 16 : 16;
  if (d->bias && 4 * 32 * p.wk * dp * (d->dtype == DP_F32 ? 4 : 2) / 1024 * 1040 + d->buckets * (NT + (int)group) * 4 + last > 163840) p.wk = 1;
  p.items = (int)(rows / (BM / p.wk) + d->nseq + 1);
  // a block of keys walks all rows that see them: the longest such walk bounds the time unless it is
  // cut. About 1024 blocks (causal order leaves half of the cuts empty), at least 512 rows each
  const int64_t kblocks = (int64_t)(d->tk / BM + 1) * d->kv_heads;
  int64_t cuts = std::min<int64_t>(16, (1024 + kblocks - 1) / kblocks * (d->causal ? 2 : 1));
  cuts = std::min(cuts, std::max<int64_t>(1, ((int64_t)1 << 30) / std::max<int64_t>(1, (int64_t)d->tk * d->kv_heads * d->dim * 8)));
  const int64_t per = std::max<int64_t>(512, ((rows + cuts - 1) / cuts + 63) / 64 * 64);
  cuts = std::min(cuts, (rows + per - 1) / per);
  int64_t tiles = d->tk / BM + d->nseq + 1;
  if (cuts > 1) {
    p.cuts = (int)cuts;
    p.cut_rows = (int)per;
    tiles = std::min(tiles * cuts, tiles + (d->tk / BM + 1) * (rows / per + 1));
  }
  p.ktiles = (int)std::min<int64_t>(tiles, INT32_MAX);
  return p;
}

static int grow_lds(const void* kern, int lds) {
  if (lds <= 65536) return 0;
  const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  DP_REQUIRE(e == hipSuccess, "dp_packed_attn_bwd: %d bytes of LDS: %s", lds, hipGetErrorString(e));
  return 0;
}

template <typename T, int DP, int WK, bool BIAS>
int launch_q(const Args& a, hipStream_t s) {
  constexpr int BN = WK > 1 ? 32 * WK : sizeof(T) == 2 ? 64 : 32;
  const int lds = 4 * Tile<T, DP>::bytes(BN) + (BIAS ? a.buckets * NT * 4 + bias_lds(a) : 0);
  const auto kern = packed_bwd_q_kernel<T, DP, WK, BN, BIAS>;
  if (const int rc = grow_lds((const void*)kern, lds)) return rc;
  hipLaunchKernelGGL(kern, dim3(a.tiles * a.hkv), dim3(NT), lds, s, a);
  return 0;
}

template <typename T, int DP, bool BIAS>
int launch(const Args& a, int wk, void* dbias, int bias_f32, hipStream_t s) {
  constexpr int BR = sizeof(T) == 2 ? 64 : 32;
  constexpr int W = sizeof(T) == 2 || DP <= 64 ? 4 : 2;
  if (a.tq > 0)
    if (const int rc = wk > 1 ? launch_q<T, DP, W, BIAS>(a, s) : launch_q<T, DP, 1, BIAS>(a, s)) return rc;
  if (a.tk > 0) {
    const int lds = 4 * Tile<T, DP>::bytes(BR) + 16 * BR * 2 + bias_lds(a);
    const auto kern = packed_bwd_kv_kernel<T, DP, BR, BIAS>;
    if (const int rc = grow_lds((const void*)kern, lds)) return rc;
    hipLaunchKernelGGL(kern, dim3(a.ktiles * a.hkv), dim3(NT), lds, s, a);
    if (a.cuts > 1) {
      const int64_t n = (int64_t)a.tk * a.hkv, per = NT / (DP / 4);
      hipLaunchKernelGGL((packed_kv_join_kernel<T, DP>), dim3((unsigned)((n + per - 1) / per)), dim3(NT), 0, s, a);
    }
  }
  if constexpr (BIAS) {
    const int tiles = a.tq > 0 ? a.tiles : 0;
    if (bias_f32)
      hipLaunchKernelGGL((packed_dbias_kernel<float>), dim3(a.hkv * a.group), dim3(NT), 0, s, (float*)dbias,
                         a.dbias_part, tiles, a.hkv, a.group, a.buckets);
    else
      hipLaunchKernelGGL((packed_dbias_kernel<T>), dim3(a.hkv * a.group), dim3(NT), 0, s, (T*)dbias, a.dbias_part,
                         tiles, a.hkv, a.group, a.buckets);
  }
  return dp_check_launch("dp_packed_attn_bwd");
}

template <typename T, bool BIAS>
int launch_dim(const Args& a, int wk, void* dbias, int bias_f32, hipStream_t s) {
  if (a.dim <= 32) return launch<T, 32, BIAS>(a, wk, dbias, bias_f32, s);
  if (a.dim <= 64) return launch<T, 64, BIAS>(a, wk, dbias, bias_f32, s);
  return launch<T, 128, BIAS>(a, wk, dbias, bias_f32, s);
}

}  // namespace

int64_t dp_packed_bwd_ws_bytes(const dp_packed_attn* d) {
  const Plan p = plan_of(d);
  int64_t n = (int64_t)d->tq * d->heads + (d->bias ? (int64_t)p.items * d->heads * d->buckets : 0);
  n = (n + 3) / 4 * 4;
  if (p.cuts > 1) n += (int64_t)d->tk * d->kv_heads * ((int64_t)p.cuts * 2 * d->dim + 1);
  return n * 4;
}

extern "C" int dp_packed_attn_bwd(const dp_packed_attn* d, void* stream) {
  Args a;
  if (const int rc = dp_packed_attn_args(d, &a, "dp_packed_attn_bwd", true)) return rc;
  DP_REQUIRE((d->lse && d->dout && d->dq) || d->tq == 0, "dp_packed_attn_bwd: no lse, dout or dq");
  DP_REQUIRE((d->dk && d->dv) || d->tk == 0, "dp_packed_attn_bwd: no dk or dv");
  DP_REQUIRE(!d->bias || d->dbias, "dp_packed_attn_bwd: no dbias");
  DP_REQUIRE(((uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv) % 16 == 0,
             "dp_packed_attn_bwd: gradients are not 16-byte aligned");
  const int64_t need = dp_packed_attn_ws_bytes(d, 1);
  DP_REQUIRE(d->ws_bytes >= need && (d->ws || !need), "dp_packed_attn_bwd: workspace holds %lld bytes, needs %lld",
             (long long)d->ws_bytes, (long long)need);
  a.dout = d->dout; a.g_row = d->g_row; a.g_head = d->g_head; a.dq = d->dq; a.dk = d->dk; a.dv = d->dv;
  const Plan p = plan_of(d);
  a.tiles = p.items;
  a.ktiles = p.ktiles;
  a.cuts = p.cuts;
  a.cut_rows = p.cut_rows;
  DP_REQUIRE((int64_t)p.ktiles * a.hkv < INT32_MAX, "dp_packed_attn_bwd: too many tiles");
  a.dsum = (float*)d->ws;
  a.dbias_part = a.dsum + (int64_t)d->tq * d->heads;
  a.kv_part = a.dsum + ((int64_t)d->tq * d->heads + (a.bias ? (int64_t)p.items * d->heads * d->buckets : 0) + 3) / 4 * 4;
  a.kv_n = (int*)(a.kv_part + (int64_t)p.cuts * a.tk * a.hkv * 2 * a.dim);
  hipStream_t s = as_stream(stream);
  const int bf = d->bias_dtype == DP_F32;
  if (d->dtype == DP_BF16)
    return a.bias ? launch_dim<bf16_t, true>(a, p.wk, d->dbias, bf, s) : launch_dim<bf16_t, false>(a, p.wk, d->dbias, bf, s);
  return a.bias ? launch_dim<float, true>(a, p.wk, d->dbias, bf, s) : launch_dim<float, false>(a, p.wk, d->dbias, bf, s);
}
