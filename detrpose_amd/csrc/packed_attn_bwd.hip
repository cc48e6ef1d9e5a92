// Attention over packed sequences, backward (packed_attn.h has the layouts).
//
//   p = exp(s - lse), dp = dO V^T, D = sum_d dO O, ds = p (dp - D)
//   dQ = scale ds K, dK = scale ds^T Q, dV = p^T dO, dbias[bucket][head] = sum of ds in the bucket
//
// Two kernels, each owner of what it writes, so nothing is added atomically and equal inputs give
// equal bits: packed_bwd_q_kernel walks the keys of a tile of 128 rows (S^T, dP^T, dQ^T: three products)
// and stores D; packed_bwd_kv_kernel walks the rows (head after head of the group, so grouped heads are summed
// in the accumulators) of a tile of 128 keys (S, dP, dV^T, dK^T: four products). Two of the seven products
// are done twice in exchange. p and ds are rounded to bf16 for their products, as p in the forward.
//
// The table's gradient comes from the first kernel: each lane owns one row (one head), so it adds its
// ds into its own LDS bins [bucket][thread] (a 4-byte add with no other lane at that address; one add
// per tile where the whole tile lies in one bucket); the block then adds the bins of a head's rows and
// writes one part per block, and packed_dbias_kernel adds the parts, all in fixed orders.
// Measured (the least of 25 launches; medians are up to 5 % above), 7055 tokens, 16 heads over 4 x 128: dq 145 us
// (850 TFLOP/s), dk / dv 240 (690) and 17 for their join; 4031 tokens, 16 over 8 x 64 with 32 buckets: 116, 64 and 10.
#include "packed_attn.h"
#include <algorithm>

int dp_packed_attn_args(const dp_packed_attn* d, dppa::Args* a, const char* what, bool backward);

namespace {
using namespace dppa;

// dk / dv: 128 keys (32 a wave, their K fragments in registers) walk over tiles of BR query rows of one head after
// the other, all heads of the group: units of work. A key tile counts group x (query tiles that see its first
// key) units and COST for its start. All key tiles of one key head, behind each other, are cut into equal shares, one
// a block, wherever the cut falls: causal order and ragged lengths leave no equal pieces otherwise (blocks of one
// tile and a bounded walk each kept 1.2 of 2 waves a SIMD busy; training at dim 128, us with such blocks and with
// shares: 7055 tokens in six sequences 588 / 490, 4096 in one 500 / 435, 32 x 512 470 / 406; at dim 64 7 k tokens 320 /
// 290, but 16 x 400 without order, equal tiles that are cut for nothing, 104 / 114). A tile that lies in several shares
// leaves parts in f32, which packed_kv_join_kernel adds in their order. Where shares would be shorter than kunits, they are
// kunits long and every tile begins a new one, so that a small call's sums do not depend on its company.
constexpr int COST = 2;

// one sequence's key tiles: tile t begins its walk at query tile clamp(t R + f, 0, q)
template <int BR>
struct Tiles {
  static constexpr int R = BM / BR;
  int n, q, f;
  bool causal;
  __device__ __forceinline__ Tiles(const Args& a, int lk, int lq)
      : n((lk + BM - 1) / BM), q((lq + BR - 1) / BR), f(-((lk - lq + (lk >= lq ? BR - 1 : 0)) / BR)), causal(a.causal) {}
  __device__ __forceinline__ int from(int t) const {
    return causal ? (int)min(max((int64_t)t * R + f, (int64_t)0), (int64_t)q) : 0;
  }
  __device__ __forceinline__ int64_t units(int group, int t) const { return (int64_t)group * (q - from(t)) + COST; }
  // of the first m tiles: all walks whole, less an arithmetic series where they begin later
  __device__ __forceinline__ int64_t sum(int group, int64_t m) const {
    int64_t late = 0;
    if (causal) {
      const int64_t t1 = min(m, (int64_t)(f > 0 ? 0 : -f / R + 1));                        // the first that begins later
      const int64_t t2 = min(m, max(t1, (int64_t)(q > f ? ((int64_t)q - f + R - 1) / R : 0)));   // that has no walk
      late = (t2 - t1) * f + R * ((t1 + t2 - 1) * (t2 - t1) / 2) + (m - t2) * q;
    }
    return m * ((int64_t)group * q + COST) - group * late;
  }
  __device__ __forceinline__ int64_t sum_in_shares(int group, int share) const {
    int64_t s = 0;
    for (int t = 0; t < n; ++t) s += (units(group, t) + share - 1) / share;
    return s * share;
  }
};

__device__ __forceinline__ int64_t lane_value(int64_t x, int l) { return __shfl((long long)x, l, 64); }

template <int BR, typename VISIT>
__device__ __forceinline__ void each_64(const Args& a, VISIT visit) {   // visit(first sequence, lane's starts and lengths)
  const int lane = threadIdx.x & 63;
  for (int base = 0; base <= a.nseq; base += 64) {   // the rows behind the last sequence are one more
    const int b = base + lane;
    int k0 = 0, lk = 0, q0 = 0, lq = 0;
    if (b <= a.nseq && a.nseq) {
      const int c0 = a.cu_k[b], c1 = a.cu_k[min(b + 1, a.nseq)], d0 = a.cu_q[b], d1 = a.cu_q[min(b + 1, a.nseq)];
      k0 = b ? clampi(c0, 0, a.tk) : 0;
      lk = max(0, (b < a.nseq ? clampi(c1, 0, a.tk) : a.tk) - k0);
      q0 = b && b < a.nseq ? clampi(d0, 0, a.tq) : 0;
      lq = b < a.nseq ? max(0, clampi(d1, 0, a.tq) - q0) : 0;
    } else if (b == 0) {
      lk = a.tk;   // no sequences
    }
    if (!visit(base, k0, lk, q0, lq)) return;
  }
}

template <int BR>
__device__ __forceinline__ int64_t total_units(const Args& a) {
  int64_t all = 0;
  each_64<BR>(a, [&](int, int, int lk, int, int lq) {
    const Tiles<BR> ts(a, lk, lq);
    int64_t x = lk ? ts.sum(a.group, ts.n) : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor((long long)x, o, 64);
    all += x;
    return true;
  });
  return all;
}

// what begins at unit pos of a share that ends at unit end: tile number `at` of all, its units [u0, u1) of w
struct Found { int start, len, start2, len2, tile, at, parts; int64_t u0, u1, w; };

template <int BR>
__device__ __forceinline__ bool find_piece(const Args& a, int64_t pos, int64_t end, int64_t share, bool own, Found& out) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  int tiles = 0;
  bool found = false;
  Found p{};
  each_64<BR>(a, [&](int, int k0, int lk, int q0, int lq) {
    const Tiles<BR> ts(a, lk, lq);
    const int64_t mine = !lk ? 0 : own ? ts.sum_in_shares(a.group, (int)share) : ts.sum(a.group, ts.n);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t u = __shfl_up((long long)upto, o, 64);
      if (lane >= o) upto += u;
    }
    int count = lk ? ts.n : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(count, o, 64);
      if (lane >= o) count += u;
    }
    const int64_t all = lane_value(upto, 63);
    if (pos >= before + all) {
      before += all;
      tiles += __shfl(count, 63, 64);
      return true;
    }
    const int l = __ffsll((long long)__ballot(pos < before + upto)) - 1;
    p.start = __shfl(k0, l, 64);
    p.len = __shfl(lk, l, 64);
    p.start2 = __shfl(q0, l, 64);
    p.len2 = __shfl(lq, l, 64);
    int64_t x = pos - before - lane_value(upto - mine, l);
    const Tiles<BR> s(a, p.len, p.len2);
    if (own) {
      for (p.tile = 0; p.tile < s.n - 1; ++p.tile) {
        const int64_t w = (s.units(a.group, p.tile) + share - 1) / share * share;
        if (x < w) break;
        x -= w;
      }
    } else {
      int lo = 0, hi = s.n - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.sum(a.group, mid) <= x) lo = mid;
        else hi = mid - 1;
      }
      p.tile = lo;
      x -= s.sum(a.group, lo);
    }
    p.u0 = x;
    p.w = s.units(a.group, p.tile);
    p.u1 = min(p.w, p.u0 + end - pos);
    const int64_t at = pos - x;   // where the tile begins
    p.at = tiles + __shfl(count, l, 64) - s.n + p.tile;
    p.parts = (int)((at + p.w - 1) / share - at / share) + 1;
    found = true;
    return false;
  });
  out = p;
  return found;
}

// The pieces of every share, a wave a share, found by blocks of the dq kernel beside its own: kv_share[r] = the first and last of share r's. Piece number = share + tile
// of all tiles, which rises from piece to piece, with a gap where a tile begins with a share. (In the kernel that
// walks, the search's scalars cost 45 registers a wave.)
template <int BR>
__device__ __forceinline__ void plan_share(const Args& a, int r) {
  const int lane = threadIdx.x & 63;
  if (r >= a.kshares) return;
  const int64_t total = total_units<BR>(a);
  const bool own = total <= (int64_t)a.kblocks * a.kunits;   // every tile begins a share
  const int64_t share = own ? a.kunits : (total + a.kblocks - 1) / a.kblocks, end = (r + 1) * share;
  int lo = 0, hi = -1;
  for (int64_t pos = r * share; pos < end;) {
    Found f;
    if (!find_piece<BR>(a, pos, end, share, own, f)) break;
    const int at = own ? r : r + f.at;
    // at most two tiles of a share are not whole: the one that the share begins in, and the one that begins in it
    const int place = own ? r : 2 * r + (f.u0 == 0);
    if (at >= a.kpieces || (f.parts > 1 && place >= a.kslots)) break;   // offsets that do not rise
    const int64_t walk = f.w - COST;
    int64_t w0 = min(f.u0, walk), w1 = min(f.u1, walk);
    if (own) {   // a tile's shares alike
      const int64_t step = (walk + f.parts - 1) / f.parts;
      w0 = min(f.u0 / share * step, walk);
      w1 = min(w0 + step, walk);
    }
    if (lane == 0)
      a.kv_piece[at] = Piece{f.start, f.len, f.start2, f.len2, f.tile, (int)w0, (int)w1, own ? -f.parts : f.parts,
                             f.u0 == 0, place * BM, {0, 0}};
    if (hi < 0) lo = at;
    hi = at;
    pos = own ? end : pos + f.u1 - f.u0;
  }
  if (lane == 0) a.kv_share[r] = int2{lo, hi};
}

// WK waves of a block share its rows and take the key tile's subtiles in turn, as in the forward
template <typename T, int DP, int WK, int BN, bool BIAS>
__global__ __launch_bounds__(NT)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && DP == 128 ? 1 : 2, DP == 128 ? 2 : 8))) void packed_bwd_q_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int TB = TL::bytes(BN), NS = BN / 32 / WK, ROWS = BM / WK, OP = DP + 4;
  static_assert(WK == 1 || 4 * TB >= 4 * 32 * OP * 4, "the join of the waves fits the tiles");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform: scalar branches below
  if ((int)blockIdx.x >= a.tiles * a.hkv) {
    plan_share<sizeof(T) == 2 && DP < 128 ? 64 : 32>(a, (blockIdx.x - a.tiles * a.hkv) * (NT / 64) + wave);
    return;
  }
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
    if constexpr (sizeof(T) == 2) {
      if (a.out_lo) {
        load_frags<T, DP>(a.out_lo + at * a.dim, ok, a.dim, h, of);
#pragma unroll
        for (int s = 0; s < TL::KS; ++s) {
          const T* x = reinterpret_cast<const T*>(&of[s]);
          const T* y = reinterpret_cast<const T*>(&gf[s]);
#pragma unroll
          for (int e = 0; e < TL::VN; ++e) D = fmaf(to_f32(x[e]), to_f32(y[e]), D);
        }
      }
    }
    D = half_sum(D);
  }
  if (ok && h == 0 && wk == 0) a.dsum[at] = D;
  const float lse = ok ? a.lse[at] : INFINITY, lse_lo = BIAS && ok && a.lse_lo ? a.lse_lo[at] : 0.f;

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
        const float p = __builtin_amdgcn_exp2f(BIAS ? fmaf(s[i] - lse, LOG2E, -lse_lo) : fmaf(s[i], c, -lse));
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

template <typename T, int DP, int BR, bool BIAS>
__global__ __launch_bounds__(NT, sizeof(T) == 2 ? 2 : 1) void packed_bwd_kv_kernel(const Args a) {
  using TL = Tile<T, DP>;
  constexpr int TB = TL::bytes(BR), NS = BR / 32;
  // bf16 at dim 128: dk, dv and the K fragments take 160 of a wave's 256 registers; V's stay in LDS (with
  // them in registers 11 to 34 spilled, and each reload waited for the tile loads in flight)
  constexpr bool VL = sizeof(T) == 2 && DP == 128;
  constexpr int VB = VL ? TL::bytes(BM) : 0;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* const vtile = smem + 4 * TB;
  // lse and D of a tile's rows, and lse_lo with a bias, two buffers
  constexpr int STATS = BIAS ? 3 : 2;
  float* lse_s = reinterpret_cast<float*>(vtile + VB);
  float *dsum_s = lse_s + 2 * BR, *lo_s = dsum_s + 2 * BR;
  const int wave = uniform(threadIdx.x >> 6);   // uniform: scalar branches below
  const int kvh = uniform(blockIdx.x % a.hkv);
  const int heads = a.hkv * a.group;
  Bias bias{};
  if constexpr (BIAS) bias = bias_setup<T>(a, vtile + VB + 8 * STATS * BR, kvh);
  const int2 run = a.kv_share[blockIdx.x / a.hkv];
  const int begin = uniform(run.x), last = uniform(run.y);
  for (int piece = begin; piece <= last; ++piece) {
    const Piece pc = a.kv_piece[piece];
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // what depends on it is computed for each piece
    const int h = lane >> 5;
    const int k0 = uniform(pc.start), lk = uniform(pc.len), q0 = uniform(pc.start2), lq = uniform(pc.len2), tile = uniform(pc.tile);
    const int off = lk - lq, qtiles = (lq + BR - 1) / BR;
    const int first = tile * BM + 32 * wave, key = first + (lane & 31);
    const bool ok = key < lk;
    // the first query that sees a key
    auto sees = [&](int kk) { return a.causal ? max(0, kk - off) : 0; };
    const int mine = ok ? sees(key) : lq, wfirst = uniform(sees(first)), wlast = uniform(sees(min(first + 31, lk - 1)));
    const unsigned seen = (unsigned)max(0, lq - mine);
    // this piece's run of the walk
    const int from = uniform(min(sees(tile * BM) / BR, qtiles)), nper = qtiles - from;
    const int w0 = uniform(pc.w0), w1 = uniform(pc.w1), parts = uniform(pc.parts);
    const int begins = uniform(pc.begins), place = uniform(pc.row);
    if (piece > begin) __syncthreads();   // the tiles of the piece before are read

    u32x4 kf[TL::KS], vf[VL ? 1 : TL::KS];
    load_frags<T, DP>((const T*)a.k + (int64_t)(k0 + min(key, lk - 1)) * a.k_row + kvh * a.k_head, ok, a.dim, h, kf);
    if constexpr (VL) {
      const int vs = (int)(a.v_row * sizeof(T));
      stage_rows<T, DP, BM>((const T*)a.v + (int64_t)(k0 + tile * BM) * a.v_row + kvh * a.v_head, vs, lk - tile * BM, vtile,
                            a.dim, lane_off<T, DP>(vs, a.dim), wave);
    } else {
      load_frags<T, DP>((const T*)a.v + (int64_t)(k0 + min(key, lk - 1)) * a.v_row + kvh * a.v_head, ok, a.dim, h, vf);
    }

    const int qs = (int)(a.q_row * sizeof(T)), gs = (int)(a.g_row * sizeof(T));
    const int qoff = lane_off<T, DP>(qs, a.dim), goff = lane_off<T, DP>(gs, a.dim);
    auto fetch = [&](int buf, int g, int t) {
      char* at = smem + buf * 2 * TB;
      const int p0 = t * BR, left = lq - p0, head = kvh * a.group + g;
      stage_rows<T, DP, BR>((const T*)a.q + (int64_t)(q0 + p0) * a.q_row + head * a.q_head, qs, left, at, a.dim, qoff, wave);
      stage_rows<T, DP, BR>((const T*)a.dout + (int64_t)(q0 + p0) * a.g_row + head * a.g_head, gs, left, at + TB, a.dim,
                            goff, wave);
      // the first waves: lse, D and lse_lo, one row a lane (0 past the sequence, where q, dout and p are 0 too, and
      // where there is no lse_lo)
      if (wave < STATS) {
        const bool none = wave == 2 && !a.lse_lo;
        const float* stat = wave == 1 ? a.dsum : wave == 2 && !none ? a.lse_lo : a.lse;
        const i32x4 rs = make_rsrc(stat + (int64_t)(q0 + p0) * heads + head);
        dma4(rs, reinterpret_cast<char*>(lse_s + wave * 2 * BR + buf * BR),
             lane < min(left, BR) && !none ? lane * heads * 4 : OOB, BR);
      }
    };

    const float c = a.scale * LOG2E;
    f32x16 dk[TL::ND], dv[TL::ND];
#pragma unroll
    for (int t = 0; t < TL::ND; ++t) dk[t] = dv[t] = zero16();

    dpconv::wait_vmcnt<0>();   // the fragments above, so that the loop's waits count tiles only
    int g = uniform(nper ? w0 / nper : 0), t = uniform(from + w0 - g * nper);
    if (w0 < w1) fetch(0, g, t);
    for (int w = w0; w < w1; ++w) {
      tile_barrier();
      const int b = (w - w0) & 1, p0 = t * BR, gh = g;
      const bool turn = t + 1 == qtiles;
      t = uniform(turn ? from : t + 1);
      g = uniform(turn ? g + 1 : g);
      if (w + 1 < w1) fetch(b ^ 1, g, t);
      const char* buf = smem + b * 2 * TB;
      if (first >= lk) continue;
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        const int p32 = p0 + 32 * u;
        if (p32 >= lq) break;
        if (p32 + 31 < wfirst) continue;
        f32x16 s = rows_mma<T, DP>(buf, u, lane, kf);
        if constexpr (BIAS) {
          const float* tab = bias.tab + gh * bias.nb;
          const int rel0 = key - off - p32 - 4 * h;
          const int one = bias.one_bucket(first - min(p32 + 31, lq - 1) - off, first + 31 - p32 - off);
          if (one >= 0) {
            const float x = tab[one];
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], a.scale, x);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], a.scale, tab[bias.bucket(rel0 - 8 * (i / 4) - (i & 3))]);
          }
        }
        const int x0 = b * BR + 32 * u + 4 * h;
        const bool edge = p32 < wlast || p32 + 32 > lq || first + 32 > lk;
        // queries [mine, lq) see the key: one comparison each
        auto hidden = [&](int i) { return (unsigned)(p32 + 8 * (i / 4) + 4 * h + (i & 3) - mine) >= seen; };
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(lse_s + x0 + 8 * e);
          f32x4 lo;
          if constexpr (BIAS) lo = *reinterpret_cast<const f32x4*>(lo_s + x0 + 8 * e);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = s[4 * e + i];
            s[4 * e + i] = __builtin_amdgcn_exp2f(BIAS ? fmaf(v - ls[i], LOG2E, -lo[i]) : fmaf(v, c, -ls[i]));
          }
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (hidden(i)) s[i] = 0.f;
        }
        cols_mma<T, DP>(buf + TB, u, lane, s, dv);
        f32x16 dp;
        if constexpr (VL) {
          const RowReader<T, DP> gr(buf + TB + TL::bytes(32) * u, lane), vr(vtile + TL::bytes(32) * wave, lane);
          dp = zero16();
#pragma unroll
          for (int q = 0; q < TL::KS; ++q)
            dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(gr.read(0, q), vr.read(0, q), dp, 0, 0, 0);
        } else {
          dp = rows_mma<T, DP>(buf + TB, u, lane, vf);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f32x4 dd = *reinterpret_cast<const f32x4*>(dsum_s + x0 + 8 * e);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[4 * e + i] *= dp[4 * e + i] - dd[i];
        }
        if (edge) {   // dout of a hidden query may be anything
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (hidden(i)) s[i] = 0.f;
        }
        cols_mma<T, DP>(buf, u, lane, s, dk);
      }
    }

    if (ok) {
      const int64_t kr = (int64_t)(k0 + key) * a.hkv + kvh;
      const int row = kvh * a.kslots * BM + place + 32 * wave + (lane & 31);
      float* part = a.kv_part + (int64_t)row * 2 * a.dim;
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
            if (abs(parts) > 1) {
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
      if (begins && h == 0) a.kv_n[kr] = int2{parts, row};   // 1 part: the result is written
    }
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
  const int2 p = a.kv_n[kr];
  const int n = abs(p.x), most = a.hkv * a.kslots * BM;
  if (n <= 1) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll 4
  for (int c = 0; c < n; ++c) {
    const int row = p.y + (p.x < 0 ? c : max(0, 2 * c - 1)) * BM;   // places of shares in turn, or every other one
    if (row < 0 || row >= most) break;
    const float* part = a.kv_part + (int64_t)row * 2 * a.dim + d;
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
constexpr int KV_BLOCKS = 512;
struct Plan { int wk, items, kunits, kblocks, kslots, kshares, kpieces; };
static Plan plan_of(const dp_packed_attn* d) {
  const int64_t group = d->heads / d->kv_heads, rows = d->tq * group, seqs = std::max(1, d->nseq);
  Plan p{1, 0, 0, 1, 0};
  const int64_t wide = (rows / BM + 1) * d->kv_heads;
  if (wide < 256 && d->tk <= 2048 * seqs) p.wk = d->dtype == DP_F32 && d->dim > 64 ? 2 : 4;
  // the bins beside the waves' larger key tile: where both do not fit the LDS, the waves lie along the rows
  const int dp = d->dim <= 32 ? 32 : d->dim <= 64 ? 64 : 128, last = d->bias && d->buckets > 2 ? 4096 + 16 : 16;
  if (d->bias && 4 * 32 * p.wk * dp * (d->dtype == DP_F32 ? 4 : 2) / 1024 * 1040 + d->buckets * (NT + (int)group) * 4 + last > 163840) p.wk = 1;
  p.items = (int)(rows / (BM / p.wk) + d->nseq + 1);
  // dk / dv: two blocks a CU are what its registers allow, so 512 shares (768 and 1024: 559 and 522 us for 490), of 256
  // rows at least (512: 146 us for 115 in f32). Where every tile begins a share, all the units together are at most
  // kblocks x kunits, so the tiles at most that over COST, and the shares one a tile more than kblocks
  const int64_t br = d->dtype == DP_F32 || d->dim > 64 ? 32 : 64;
  const int64_t tiles = d->tk / BM + d->nseq + 1, walk = group * ((d->tq + br - 1) / br) + COST;   // of a tile at most
  p.kunits = (int)(256 / br);
  p.kblocks = (int)std::min<int64_t>(std::max<int64_t>(1, KV_BLOCKS / d->kv_heads), tiles * ((walk + p.kunits - 1) / p.kunits));
  p.kshares = (int)(p.kblocks + std::min<int64_t>(tiles, (int64_t)p.kblocks * p.kunits / COST));
  p.kpieces = (int)(p.kshares + tiles);
  p.kslots = (int)std::max(2 * p.kblocks, p.kshares);
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
  hipLaunchKernelGGL(kern, dim3(a.tiles * a.hkv + (a.kshares + NT / 64 - 1) / (NT / 64)), dim3(NT), lds, s, a);
  return 0;
}

template <typename T, int DP, bool BIAS>
int launch(const Args& a, int wk, void* dbias, int bias_f32, hipStream_t s) {
  constexpr int BR = sizeof(T) == 2 && DP < 128 ? 64 : 32;
  constexpr int W = sizeof(T) == 2 || DP <= 64 ? 4 : 2;
  if (a.tq > 0 || a.tk > 0)
    if (const int rc = wk > 1 ? launch_q<T, DP, W, BIAS>(a, s) : launch_q<T, DP, 1, BIAS>(a, s)) return rc;
  if (a.tk > 0) {
    const int lds = 4 * Tile<T, DP>::bytes(BR) + (sizeof(T) == 2 && DP == 128 ? Tile<T, DP>::bytes(BM) : 0) + (BIAS ? 24 : 16) * BR + bias_lds(a);
    const auto kern = packed_bwd_kv_kernel<T, DP, BR, BIAS>;
    if (const int rc = grow_lds((const void*)kern, lds)) return rc;
    hipLaunchKernelGGL(kern, dim3(a.kshares * a.hkv), dim3(NT), lds, s, a);
    const int64_t walk = (int64_t)a.group * ((a.tq + BR - 1) / BR) + COST;   // of a tile at most
    if (walk > a.kunits || ((int64_t)a.tk / BM + a.nseq + 1) * walk > (int64_t)a.kblocks * a.kunits) {   // else no tile is cut
      const int64_t n = (int64_t)a.tk * a.hkv, per = NT / (DP / 4);
      hipLaunchKernelGGL((packed_kv_join_kernel<T, DP>), dim3((unsigned)((n + per - 1) / per)), dim3(NT), 0, s, a);
    }
  }
  if constexpr (BIAS) {
    const int tiles = a.tiles;
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
  n += (int64_t)d->kv_heads * p.kslots * BM * 2 * d->dim + (int64_t)p.kpieces * (sizeof(Piece) / 4) + (int64_t)p.kshares * 2 +
       (int64_t)d->tk * d->kv_heads * 2;
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
  a.tiles = a.tq > 0 ? p.items : 0;
  a.kblocks = p.kblocks;
  a.kunits = p.kunits;
  a.kslots = p.kslots;
  a.kshares = p.kshares;
  a.kpieces = p.kpieces;
  // every launch's grid has less than 2^32 threads; the join of dk / dv takes dp / 4 of them a key row
  const int64_t per = NT / ((a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128) / 4);
  DP_REQUIRE((int64_t)p.items * a.hkv + p.kshares <= UINT32_MAX / NT && (int64_t)p.kslots * a.hkv < INT32_MAX / BM &&
                 ((int64_t)a.tk * a.hkv + per - 1) / per <= UINT32_MAX / NT,
             "dp_packed_attn_bwd: too many tiles");
  a.dsum = (float*)d->ws;
  a.dbias_part = a.dsum + (int64_t)d->tq * d->heads;
  a.kv_part = a.dsum + ((int64_t)d->tq * d->heads + (a.bias ? (int64_t)p.items * d->heads * d->buckets : 0) + 3) / 4 * 4;
  a.kv_piece = (Piece*)(a.kv_part + (int64_t)a.hkv * p.kslots * BM * 2 * a.dim);
  a.kv_share = (int2*)(a.kv_piece + p.kpieces);
  a.kv_n = a.kv_share + p.kshares;
  hipStream_t s = as_stream(stream);
  const int bf = d->bias_dtype == DP_F32;
  if (d->dtype == DP_BF16)
    return a.bias ? launch_dim<bf16_t, true>(a, p.wk, d->dbias, bf, s) : launch_dim<bf16_t, false>(a, p.wk, d->dbias, bf, s);
  return a.bias ? launch_dim<float, true>(a, p.wk, d->dbias, bf, s) : launch_dim<float, false>(a, p.wk, d->dbias, bf, s);
}
