// Attention over packed sequences, forward (packed_attn.h has the layouts).
//
// One pass over the keys with the running maximum and sum of the softmax: a block owns 128 rows
// (query x head of the group) of one (sequence, key head), 32 a wave, and walks key tiles of BN rows,
// double-buffered in LDS. Per wave and 32 keys: S^T = K Q^T, p = exp(s - m), O^T += V^T P^T; a lane
// holds one row's scores, so the maximum needs one exchange between the wave's halves, and the sum
// none until the end. m moves only when a row's maximum grows by more than 8 in the exponent of 2
// (p stays below 256): the rescaling of O is then rare. p is rounded to bf16 for its product (by at most 2^-8
// of itself, as the output's own rounding); the sum takes it unrounded.
// Bound by the matrix pipe beside the exponentials: causal prompts of 8075 tokens, 32 heads x 128, 211 us, 870
// TFLOP/s; where rows are few by HBM: 16 single tokens over 128 k keys 124 us, 4.2 TB/s.
#include "packed_attn.h"
#include <algorithm>

namespace {
using namespace dppa;

constexpr float GROW = 8.f;   // log2 of how far p may pass 1 before m moves

// A row again, key by key: only for a wave whose result holds a NaN. In the products a key that causal order
// hides has the weight 0, but 0 x inf or NaN (its value) is NaN: here hidden keys are not read. The keys that
// share a tile with the row's last one are at most NEAR behind it; where their values are finite, the NaN is
// the row's own, and so it is where one of the first 64 scores is NaN, or one of their values in every column:
// those rows stay as they are, which keeps a model whose numbers went NaN from walking every key twice.
constexpr int NEAR = 160;   // the wave's 32 rows, the tile's 128 keys

template <typename T, typename BIASOF>
__device__ __forceinline__ void slow_row(const Args& a, int kvh, int g, int pos, int q0, int k0, int lk, int lim,
                                         BIASOF bias) {
  const int lane = threadIdx.x & 63;
  const int head = kvh * a.group + g;
  const T* q = (const T*)a.q + (int64_t)(q0 + pos) * a.q_row + head * a.q_head;
  auto value = [&](int j, int d) {
    return d < a.dim ? to_f32(((const T*)a.v + (int64_t)(k0 + j) * a.v_row + kvh * a.v_head)[d]) : 0.f;
  };
  bool hides = false;
  for (int j = lim; j < min(lk, lim + NEAR); ++j) {
    const float x = value(j, lane), y = value(j, lane + 64);
    hides |= x - x != 0.f || y - y != 0.f;
  }
  if (!__ballot(hides)) return;
  auto score = [&](int j) {
    const T* k = (const T*)a.k + (int64_t)(k0 + j) * a.k_row + kvh * a.k_head;
    float s = 0.f;
    for (int d = 0; d < a.dim; ++d) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
    return s * a.scale + bias(j);
  };
  bool n0 = lane >= a.dim, n1 = lane + 64 >= a.dim;
  for (int j = 0; j < min(lim, 64); ++j) {
    const float x = value(j, lane), y = value(j, lane + 64);
    n0 |= x != x;
    n1 |= y != y;
  }
  const float s0 = lane < lim ? score(lane) : 0.f;
  if (__ballot(s0 != s0) || __ballot(n0 && n1) == ~0ull) return;
  float m = -INFINITY;
  for (int j = lane; j < lim; j += 64) m = fmaxf(m, score(j));
  m = wave_max(m);
  const float mref = m == -INFINITY ? 0.f : m;
  float sum = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < lim; j0 += 64) {
    const float p = j0 + lane < lim ? __builtin_amdgcn_exp2f((score(j0 + lane) - mref) * LOG2E) : 0.f;
    sum += p;
    for (int u = 0; u < min(64, lim - j0); ++u) {
      const float w = __shfl(p, u, 64);
      o0 = fmaf(w, value(j0 + u, lane), o0);
      o1 = fmaf(w, value(j0 + u, lane + 64), o1);
    }
  }
  sum = wave_sum(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* o = (T*)a.out + (int64_t)(q0 + pos) * a.o_row + head * a.o_head;
  bf16_t* lo = a.out_lo ? a.out_lo + ((int64_t)(q0 + pos) * a.hkv * a.group + head) * a.dim : nullptr;
#pragma unroll
  for (int d = lane; d < 128; d += 64)
    if (d < a.dim) {
      const float x = (d == lane ? o0 : o1) * inv;
      o[d] = from_f32<T>(x);
      if (lo) lo[d] = (bf16_t)(x - to_f32(o[d]));
    }
}

// chunks that a sequence's keys are cut into, for a tile of `rows` rows
__device__ __forceinline__ int splits_of(const Args& a, int lk, int rows) {
  return a.splits <= 1 ? 1 : clampi((int)(((unsigned)lk + a.chunk - 1) / max(a.chunk, 16 * rows)), 1, a.splits);
}

// WK waves of a block share its rows and walk the key tile's subtiles in turn; 4 / WK of them, 32 rows
// each, lie along the rows.
template <typename T, int DP, int WK, int BN, bool BIAS>
__global__ __launch_bounds__(NT)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && DP == 128 ? 1 : 2, DP == 128 ? 2 : 8))) void packed_fwd_kernel(const Args a, int fill_tail) {
  using TL = Tile<T, DP>;
  constexpr int TB = TL::bytes(BN), NS = BN / 32 / WK, ROWS = BM / WK, OP = DP + 4;
  // waves that lie along the keys load what they read themselves and wait for no other
  constexpr bool OWN = WK == 4 && 64 / TL::CPR % TL::PERIOD == 0;
  constexpr int SB = TL::bytes(32 * NS);   // a wave's part of a tile
  static_assert(WK == 1 || 4 * TB >= (4 * 32 * (OP + 2) + 2 * ROWS) * 4, "the join of the waves fits the tiles");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform: scalar branches below
  const int wk = wave % WK, wr = wave / WK;
  const int kvh = uniform(blockIdx.x % a.hkv);
  auto tiles_of = [&](int len) { return (len * a.group + ROWS - 1) / ROWS; };
  auto cuts_of = [&](int lq, int lk) { return splits_of(a, lk, min(ROWS, lq * a.group)); };
  Item it;
  // the last tiles first: in causal order they have the most keys
  if (!find_item(a.cu_q, a.tq, a.cu_k, a.tk, a.nseq, fill_tail || a.splits > 1, a.tiles - 1 - blockIdx.x / a.hkv,
                 [&](int len, int keys) { return tiles_of(len) * cuts_of(len, keys); }, it))
    return;
  const int q0 = it.start, lq = it.len, k0 = it.start2, lk = it.len2;
  const int cuts = uniform(cuts_of(lq, lk)), ntile = uniform(tiles_of(lq)), cut = uniform(it.sub / ntile);
  const int off = lk - lq, rows = lq * a.group, row0 = uniform(it.sub - cut * ntile) * ROWS;
  const int first = row0 + 32 * wr, r = first + (lane & 31);
  const bool ok = r < rows;
  const int rc = min(r, rows - 1), pos = rc / a.group, g = rc - pos * a.group;
  const int heads = a.hkv * a.group;
  // this block's keys [kbeg, kend) of those that a row sees: [0, limit)
  const int step = uniform(cuts > 1 ? ((lk + cuts - 1) / cuts + BN - 1) / BN * BN : 0), kbeg = cut * step;
  auto limit = [&](int row) {
    const int n = a.causal ? clampi(min(row, rows - 1) / a.group + off + 1, 0, lk) : lk;
    return cuts > 1 ? min(n, kbeg + step) : n;
  };
  const int lim = limit(r), wmin = uniform(limit(first)), wmax = uniform(first < rows ? limit(first + 31) : 0);
  const int nt = uniform(max(0, (limit(row0 + ROWS - 1) - kbeg + BN - 1) / BN));
  // positions of the wave's first and last row
  const int pfirst = uniform(first / a.group + off), plast = uniform(min(first + 31, rows - 1) / a.group + off);
  Bias bias{};
  if constexpr (BIAS) bias = bias_setup<T>(a, smem + 4 * TB, kvh);

  u32x4 qf[TL::KS];
  load_frags<T, DP>((const T*)a.q + (int64_t)(q0 + pos) * a.q_row + (kvh * a.group + g) * a.q_head, ok, a.dim, h, qf);

  const int ks = (int)(a.k_row * sizeof(T)), vs = (int)(a.v_row * sizeof(T));
  constexpr int LT = OWN ? 64 : NT;   // threads that load together
  const int koff = lane_off<T, DP, LT>(ks, a.dim), voff = lane_off<T, DP, LT>(vs, a.dim);
  auto fetch = [&](int j) {
    char* buf = smem + (j & 1) * 2 * TB + (OWN ? wk * SB : 0);
    const int key0 = kbeg + j * BN + (OWN ? 32 * NS * wk : 0), left = lk - key0;
    if (OWN && left <= 0) return;
    constexpr int R = OWN ? 32 * NS : BN;
    stage_rows<T, DP, R, LT>((const T*)a.k + (int64_t)(k0 + key0) * a.k_row + kvh * a.k_head, ks, left, buf, a.dim, koff,
                             OWN ? 0 : wave);
    stage_rows<T, DP, R, LT>((const T*)a.v + (int64_t)(k0 + key0) * a.v_row + kvh * a.v_head, vs, left, buf + TB, a.dim,
                             voff, OWN ? 0 : wave);
  };

  // scores in units in which exp(s - m) = exp2((s - m) c): raw products, or, with a bias, scaled ones
  const float c = BIAS ? LOG2E : a.scale * LOG2E;
  float m = -INFINITY, l = 0.f;
  f32x16 o[TL::ND];
#pragma unroll
  for (int t = 0; t < TL::ND; ++t) o[t] = zero16();

  if (nt > 0) fetch(0);
  for (int j = 0; j < nt; ++j) {
    if constexpr (OWN) {
      dpconv::wait_vmcnt<0>();
      asm volatile("" ::: "memory");
    } else {
      tile_barrier();
    }
    if (j + 1 < nt) fetch(j + 1);
    const char* buf = smem + (j & 1) * 2 * TB;
    const int key0 = kbeg + j * BN + 32 * NS * wk;
    if (key0 >= wmax) continue;
    f32x16 s[NS];
    rows_mma_n<T, DP, NS>(buf, NS * wk, lane, qf, s);
    if constexpr (BIAS) {
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        const int k32 = key0 + 32 * u, one = bias.one_bucket(k32 - plast, k32 + 31 - pfirst);
        const float* tab = bias.tab + g * bias.nb;
        if (one >= 0) {
          const float b = tab[one];
#pragma unroll
          for (int i = 0; i < 16; ++i) s[u][i] = fmaf(s[u][i], a.scale, b);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[u][i] = fmaf(s[u][i], a.scale, tab[bias.bucket(k32 + 8 * (i / 4) + 4 * h + (i & 3) - pos - off)]);
        }
      }
    }
    if (key0 + 32 * NS > wmin) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * u + 8 * (i / 4) + 4 * h + (i & 3) >= lim) s[u][i] = -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    top = half_max(top);
    // (top - m) c is NaN while both are -inf: no move
    const bool move = (top - m) * c > GROW;
    if (__ballot(move)) {
      const float to = move ? top : m;
      const float alpha = move ? __builtin_amdgcn_exp2f((m - to) * c) : 1.f;
      m = to;
      l *= alpha;
#pragma unroll
      for (int t = 0; t < TL::ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
    }
    const float mref = m == -INFINITY ? 0.f : m, mc = mref * c;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NS; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // with a bias s may be the type's lowest value, whose product with c overflows: subtract first
        s[u][i] = __builtin_amdgcn_exp2f(BIAS ? (s[u][i] - mref) * c : fmaf(s[u][i], c, -mc));
        sum[i & 1] += s[u][i];
      }
      cols_mma<T, DP>(buf + TB, NS * wk + u, lane, s[u], o);
    }
    l += sum[0] + sum[1];
  }
  l = half_sum(l);

  auto head_row = [&](int p, int hd) { return (int64_t)(q0 + p) * heads + kvh * a.group + hd; };
  // four results of a row: the output, or this cut's part of it
  auto put = [&](int64_t at, int p, int hd, int d, f32x4 x) {
    if (cuts > 1) {
      *reinterpret_cast<f32x4*>(a.part + ((int64_t)cut * a.tq * heads + at) * a.dim + d) = x;
    } else {
      put4<T>((T*)a.out + (int64_t)(q0 + p) * a.o_row + (kvh * a.group + hd) * a.o_head + d,
              a.out_lo ? a.out_lo + at * a.dim + d : nullptr, x);
    }
  };
  auto lse2 = [&](float mm, float ll, float none) { return ll == 0.f ? none : mm + __log2f(ll); };
  auto put_sums = [&](int64_t at, float mm, float ll) {
    if constexpr (BIAS) {
      if (cuts > 1) {   // apart: under a large bias one number, m + log l, would round the part's size away
        a.part_m[(int64_t)cut * a.tq * heads + at] = mm;
        a.part_l[(int64_t)cut * a.tq * heads + at] = ll;
      } else {
        put_lse<BIAS>(a, at, mm, ll);
      }
    } else {
      if (cuts > 1) a.part_m[(int64_t)cut * a.tq * heads + at] = lse2(mm * c, ll, -INFINITY);
      else if (a.lse) a.lse[at] = lse2(mm * c, ll, INFINITY);
    }
    if (a.splits > 1 && cut == 0) a.part_n[at] = cuts;
  };
  const bool write = it.b < a.nseq || fill_tail;

  if constexpr (WK == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    bool bad = l != l;
    const int64_t at = head_row(pos, g);
#pragma unroll
    for (int t = 0; t < TL::ND; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[t][i] *= inv;
        bad |= o[t][i] != o[t][i];
      }
    if (ok) {
      if (write)
#pragma unroll
        for (int t = 0; t < TL::ND; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = 32 * t + 8 * e + 4 * h;
            if (d < a.dim) put(at, pos, g, d, f32x4{o[t][4 * e], o[t][4 * e + 1], o[t][4 * e + 2], o[t][4 * e + 3]});
          }
      if (h == 0) put_sums(at, m, l);
    }
    if (cuts > 1) return;   // packed_join_kernel looks for NaN
    unsigned long long redo = __ballot(bad && ok);
    redo |= redo >> 32;
    for (unsigned left = (unsigned)redo; left; left &= left - 1) {
      const int row = first + __builtin_ctz(left), rp = row / a.group;
      const int hd = row - rp * a.group;
      slow_row<T>(a, kvh, hd, rp, q0, k0, lk, limit(row), [&](int j) {
        return BIAS ? bias.tab[hd * bias.nb + bias.bucket(j - rp - off)] : 0.f;
      });
    }
  } else {
    // join the WK waves of each 32 rows through LDS
    __syncthreads();
    float* oo = reinterpret_cast<float*>(smem);
    float *mm = oo + 4 * 32 * OP, *ll = mm + 128;
    int* redo = reinterpret_cast<int*>(ll + 128);
    const int x = wave * 32 + (lane & 31);
#pragma unroll
    for (int t = 0; t < TL::ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(oo + x * OP + 32 * t + 8 * e + 4 * h) =
            f32x4{o[t][4 * e], o[t][4 * e + 1], o[t][4 * e + 2], o[t][4 * e + 3]};
    if (h == 0) {
      mm[x] = m;
      ll[x] = l;
    }
    if (threadIdx.x < ROWS) redo[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * (DP / 4); i += NT) {
      const int jr = i / (DP / 4), d = (i - jr * (DP / 4)) * 4, row = row0 + jr;
      if (row >= rows || d >= a.dim) continue;
      const int w0 = (jr >> 5) * WK * 32 + (jr & 31), rp = row / a.group, hd = row - rp * a.group;
      float top = mm[w0];
#pragma unroll
      for (int w = 1; w < WK; ++w) top = fmaxf(top, mm[w0 + 32 * w]);
      const float ref = top == -INFINITY ? 0.f : top;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float tot = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float f = __builtin_amdgcn_exp2f((mm[w0 + 32 * w] - ref) * c);
        tot = fmaf(ll[w0 + 32 * w], f, tot);
        const f32x4 v = *reinterpret_cast<const f32x4*>(oo + (w0 + 32 * w) * OP + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(v[e], f, sum[e]);
      }
      const float inv = tot == 0.f ? 0.f : 1.f / tot;
      bool bad = tot != tot;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sum[e] *= inv;
        bad |= sum[e] != sum[e];
      }
      const int64_t at = head_row(rp, hd);
      if (write) put(at, rp, hd, d, sum);
      if (d == 0) put_sums(at, top, tot);
      if (bad) redo[jr] = 1;
    }
    if (cuts > 1) return;
    __syncthreads();
    for (int jr = wave; jr < min(ROWS, rows - row0); jr += 4) {
      if (!redo[jr]) continue;
      const int row = row0 + jr, rp = row / a.group;
      const int hd = row - rp * a.group;
      slow_row<T>(a, kvh, hd, rp, q0, k0, lk, limit(row), [&](int j) {
        return BIAS ? bias.tab[hd * bias.nb + bias.bucket(j - rp - off)] : 0.f;
      });
    }
  }
}

// slow_row of a row of the packed queries (its sequence is searched)
template <typename T>
__device__ __forceinline__ void redo_row(const Args& a, int row, int head) {
  int b = 0;
  while (b < a.nseq && clampi(a.cu_q[b + 1], 0, a.tq) <= row) ++b;
  if (b == a.nseq) return;
  const int2 qs = seq_at(a.cu_q, a.nseq, a.tq, b), ks = seq_at(a.cu_k, a.nseq, a.tk, b);
  const int pos = row - qs.x, off = ks.y - qs.y;
  slow_row<T>(a, head / a.group, head % a.group, pos, qs.x, ks.x, ks.y, a.causal ? clampi(pos + off + 1, 0, ks.y) : ks.y,
              [&](int j) {
                if (!a.bias) return 0.f;
                const int rel = j - pos - off, n = a.both ? abs(rel) : max(-rel, 0);
                int bk = a.both && rel > 0 ? a.buckets / 2 : 0;
                for (int e = 0; e < a.nedge; ++e) bk += a.edge[e] <= n;
                const int64_t x = (int64_t)bk * a.hkv * a.group + head;
                return a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[x]
                                  : to_f32(reinterpret_cast<const T*>(a.bias)[x]);
              });
}

// rows whose keys were cut: out = sum of the parts weighted by l exp(m - the largest m) (without a bias m holds
// m + log l, and l is 1), four elements a thread, in the order of the cuts
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(NT) void packed_join_kernel(const Args a) {
  constexpr int TPR = DP / 4;   // threads of a row
  const int heads = a.hkv * a.group;
  const int64_t all = (int64_t)a.tq * heads;
  const int64_t at = (int64_t)blockIdx.x * (NT / TPR) + threadIdx.x / TPR;
  const int d = (threadIdx.x % TPR) * 4;
  const int n = at < all ? min(a.part_n[at], a.splits) : 1;
  bool bad = false;
  if (n > 1) {
    float top = -INFINITY;
    for (int i = 0; i < n; ++i) top = fmaxf(top, a.part_m[i * all + at]);
    const float ref = top == -INFINITY ? 0.f : top;
    float tot = 0.f;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float x = (a.part_m[i * all + at] - ref) * (BIAS ? LOG2E : 1.f);
      const float f = __builtin_amdgcn_exp2f(x) * (BIAS ? a.part_l[i * all + at] : 1.f);   // a part that saw nothing: 0
      tot += f;
      if (d < a.dim) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + (i * all + at) * a.dim + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = fmaf(v[e], f, sum[e]);
      }
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
    bad = tot != tot;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum[e] *= inv;
      bad |= sum[e] != sum[e];
    }
    if (d < a.dim) {
      const int64_t row = at / heads;
      put4<T>((T*)a.out + row * a.o_row + (at - row * heads) * a.o_head + d,
              a.out_lo ? a.out_lo + at * a.dim + d : nullptr, sum);
    }
    if (d == 0) put_lse<BIAS>(a, at, ref, tot);
  }
  if (!__ballot(bad)) return;
  // NaN: the wave's rows one by one (each wave for itself: no barrier past this point but its own)
  const int lane = threadIdx.x & 63;
  for (int rr = 0; rr < 64 / TPR; ++rr) {
    const bool mine = lane / TPR == rr;
    if (!__ballot(bad && mine)) continue;
    const int64_t row_at = (int64_t)blockIdx.x * (NT / TPR) + (threadIdx.x >> 6) * (64 / TPR) + rr;
    const int row = (int)(row_at / heads);
    redo_row<T>(a, row, (int)(row_at - (int64_t)row * heads));
  }
}

// The same for few rows of many parts (single tokens over long caches): a block per row, DP / 4 lanes a
// part, and the block's 256 / (DP / 4) groups of lanes take parts in turn; summed in a fixed order.
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(NT) void packed_join_row_kernel(const Args a) {
  constexpr int TPR = DP / 4, GROUPS = NT / TPR;
  __shared__ f32x4 sm[NT];
  const int heads = a.hkv * a.group, lane = threadIdx.x & 63;
  const int64_t all = (int64_t)a.tq * heads, at = blockIdx.x;
  const int n = uniform(min(a.part_n[at], a.splits));
  if (n <= 1) return;
  const float x = lane < n ? a.part_m[lane * all + at] : -INFINITY;
  const float l = !BIAS ? 1.f : lane < n ? a.part_l[lane * all + at] : 0.f;
  const float top = wave_max(x), ref = top == -INFINITY ? 0.f : top;
  const float f = __builtin_amdgcn_exp2f((x - ref) * (BIAS ? LOG2E : 1.f)) * l, tot = wave_sum(f);
  const int grp = threadIdx.x / TPR, d = (threadIdx.x % TPR) * 4;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = grp; i < (n + GROUPS - 1) / GROUPS * GROUPS; i += GROUPS) {
    const float w = __shfl(f, i & 63, 64);   // 0 past the parts
    if (i < n && d < a.dim) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + (i * all + at) * a.dim + d);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(v[e], w, sum[e]);
    }
  }
  sm[threadIdx.x] = sum;
  __syncthreads();
  const float inv = tot == 0.f ? 0.f : 1.f / tot;
  bool bad = tot != tot;
  const int row = (int)(at / heads), head = (int)(at - (int64_t)row * heads);
  if (threadIdx.x < TPR && d < a.dim) {
#pragma unroll
    for (int k = 1; k < GROUPS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += sm[k * TPR + threadIdx.x][e];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum[e] *= inv;
      bad |= sum[e] != sum[e];
    }
    put4<T>((T*)a.out + (int64_t)row * a.o_row + head * a.o_head + d, a.out_lo ? a.out_lo + at * a.dim + d : nullptr, sum);
    if (d == 0) put_lse<BIAS>(a, at, ref, tot);
  }
  if (threadIdx.x < 64 && __ballot(bad)) redo_row<T>(a, row, head);
}

// Which shape a call runs in. Lengths are on the device, so the rule goes by totals.
struct Plan { int wk, chunk, splits, items; };
static Plan plan_of(const dp_packed_attn* d) {
  const int64_t group = d->heads / d->kv_heads, rows = d->tq * group, seqs = std::max(1, d->nseq);
  Plan p{1, 0, 1, 0};
  const int64_t wide = (rows / BM + 1) * d->kv_heads;   // blocks at least
  const bool few = rows <= 32 * seqs;
  if (few || (wide < 256 && d->tk <= 2048 * seqs)) p.wk = d->dtype == DP_F32 && d->dim > 64 ? 2 : 4;
  const int per = BM / p.wk;
  int64_t items = rows / per + d->nseq + 1;
  if (d->tk > 1024 && (few || (rows / per + 1) * d->kv_heads < 256) && d->tq > 0) {
    // about 256 blocks of few rows (a block's start costs as much as 20 tiles: 64 sequences of 2000 keys 80 us with
    // 1024 blocks, 62 with 512, 57 with 256; 128 k ragged keys 139, 130, 133), or 512 of many; a part of the output
    // is written in f32 per cut and row, so a cut has at least 16 keys a row (splits_of)
    const int64_t target = few ? 256 : 512;
    const int64_t most_tiles = rows / per + 1;             // of one sequence
    int64_t chunk = std::max<int64_t>(256, (int64_t)d->tk * d->kv_heads * (few ? 1 : (items + seqs) / seqs) / target);
    chunk = (chunk + 127) / 128 * 128;
    int64_t splits = std::min<int64_t>(64, (d->tk + chunk - 1) / chunk);
    splits = std::min(splits, std::max<int64_t>(1, (few ? 64 : 4) * target / std::max<int64_t>(1, rows / per * d->kv_heads)));
    splits = std::min(splits, std::max<int64_t>(1, ((int64_t)256 << 20) / ((int64_t)d->tq * d->heads * (d->dim + 1) * 4)));
    if (splits > 1) {
      p.chunk = (int)chunk;
      p.splits = (int)splits;
      // sum of tiles x cuts: cuts <= splits, and <= 1 + keys / chunk
      items = std::min(items * splits, items + most_tiles * (d->tk / chunk + 1));
    }
  }
  p.items = (int)std::min<int64_t>(items, INT32_MAX);
  return p;
}

template <typename T, int DP, int WK, bool BIAS>
int launch(const Args& a, int fill_tail, hipStream_t s) {
  constexpr int BN = WK > 1 ? 32 * WK : sizeof(T) == 2 ? 64 : 32;
  const int lds = 4 * Tile<T, DP>::bytes(BN) + bias_lds(a);
  const auto kern = packed_fwd_kernel<T, DP, WK, BN, BIAS>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    DP_REQUIRE(e == hipSuccess, "dp_packed_attn_fwd: %d bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, dim3(a.tiles * a.hkv), dim3(NT), lds, s, a, fill_tail);
  if (a.splits > 1) {
    const int64_t n = (int64_t)a.tq * a.hkv * a.group, per = NT / (DP / 4);
    if (n <= 4096)
      hipLaunchKernelGGL((packed_join_row_kernel<T, DP, BIAS>), dim3((unsigned)n), dim3(NT), 0, s, a);
    else
      hipLaunchKernelGGL((packed_join_kernel<T, DP, BIAS>), dim3((unsigned)((n + per - 1) / per)), dim3(NT), 0, s, a);
  }
  return dp_check_launch("dp_packed_attn_fwd");
}

template <typename T, bool BIAS>
int launch_dim(const Args& a, int wk, int fill_tail, hipStream_t s) {
  constexpr int W128 = sizeof(T) == 2 ? 4 : 2;
  if (a.dim <= 32) return wk > 1 ? launch<T, 32, 4, BIAS>(a, fill_tail, s) : launch<T, 32, 1, BIAS>(a, fill_tail, s);
  if (a.dim <= 64) return wk > 1 ? launch<T, 64, 4, BIAS>(a, fill_tail, s) : launch<T, 64, 1, BIAS>(a, fill_tail, s);
  return wk > 1 ? launch<T, 128, W128, BIAS>(a, fill_tail, s) : launch<T, 128, 1, BIAS>(a, fill_tail, s);
}

}  // namespace


int64_t dp_packed_bwd_ws_bytes(const dp_packed_attn* d);   // packed_attn_bwd.hip

extern "C" int64_t dp_packed_attn_ws_bytes(const dp_packed_attn* d, int32_t backward) {
  if (!d || d->heads <= 0 || d->kv_heads <= 0 || d->tq < 0 || d->tk < 0 || d->nseq < 0) return 0;
  if (!backward) {
    const Plan p = plan_of(d);
    return p.splits > 1 ? (int64_t)d->tq * d->heads * (p.splits * ((int64_t)d->dim + (d->bias ? 2 : 1)) + 1) * 4 : 0;
  }
  return dp_packed_bwd_ws_bytes(d);
}

// the checks that forward and backward share, and the kernels' form of the descriptor
int dp_packed_attn_args(const dp_packed_attn* d, dppa::Args* a, const char* what, bool backward) {
  DP_REQUIRE(d && d->nseq >= 0 && d->tq >= 0 && d->tk >= 0, "%s: bad arguments", what);
  DP_REQUIRE(d->dtype == DP_F32 || d->dtype == DP_BF16, "%s: dtype %d", what, d->dtype);
  DP_REQUIRE(d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0, "%s: %d heads over %d key heads", what,
             d->heads, d->kv_heads);
  DP_REQUIRE(d->dim > 0 && d->dim <= 128 && d->dim % 8 == 0, "%s: head dim %d (multiples of 8 up to 128)", what, d->dim);
  DP_REQUIRE(d->scale > 0.f && d->scale < INFINITY, "%s: scale %g", what, (double)d->scale);
  DP_REQUIRE((int64_t)d->tq * d->heads < INT32_MAX - BM && (int64_t)d->tk < INT32_MAX - BM, "%s: too many rows", what);
  // without sequences too: queries are searched for behind the last offset
  DP_REQUIRE((d->cu_q && d->cu_k) || (d->nseq == 0 && d->tq == 0), "%s: no sequence offsets", what);
  DP_REQUIRE((d->q && d->out) || d->tq == 0, "%s: no queries or output", what);
  DP_REQUIRE((d->k && d->v) || d->tk == 0, "%s: no keys or values", what);
  DP_REQUIRE(!d->out_lo || (d->dtype == DP_BF16 && d->lse && (uintptr_t)d->out_lo % 16 == 0),
             "%s: out_lo goes with bf16 and lse, 16-byte aligned", what);
  DP_REQUIRE(!d->lse_lo || d->lse, "%s: lse_lo goes with lse", what);
  const int e = d->dtype == DP_BF16 ? 2 : 4;
  struct { const char* name; const void* p; int64_t row, head; } t[] = {
      {"q", d->q, d->q_row, d->q_head}, {"k", d->k, d->k_row, d->k_head}, {"v", d->v, d->v_row, d->v_head},
      {"out", d->out, d->o_row, d->o_head}, {"dout", d->dout, d->g_row, d->g_head}};
  for (int i = 0; i < (backward ? 5 : 4); ++i) {
    DP_REQUIRE(((uintptr_t)t[i].p | (uintptr_t)(t[i].row * e) | (uintptr_t)(t[i].head * e)) % 16 == 0,
               "%s: rows of %s are not 16-byte aligned", what, t[i].name);
    // 64 rows and a group's heads are addressed from one base in 31 bits
    DP_REQUIRE(t[i].row >= 0 && t[i].head >= 0 && t[i].row * e < (1 << 24) &&
                   t[i].head * e * (d->heads / d->kv_heads) < (1 << 28),
               "%s: strides of %s too large", what, t[i].name);
  }
  *a = dppa::Args{};
  a->q = d->q; a->k = d->k; a->v = d->v; a->out = d->out; a->lse = d->lse; a->out_lo = (bf16_t*)d->out_lo;
  a->q_row = d->q_row; a->q_head = d->q_head; a->k_row = d->k_row; a->k_head = d->k_head;
  a->v_row = d->v_row; a->v_head = d->v_head; a->o_row = d->o_row; a->o_head = d->o_head;
  a->cu_q = d->cu_q; a->cu_k = d->cu_k; a->nseq = d->nseq; a->tq = d->tq; a->tk = d->tk;
  a->hkv = d->kv_heads; a->group = d->heads / d->kv_heads; a->dim = d->dim; a->causal = d->causal; a->scale = d->scale;
  if (d->bias) {
    const int nb = d->both ? d->buckets / 2 : d->buckets;
    DP_REQUIRE(d->bias_dtype == DP_F32 || d->bias_dtype == d->dtype, "%s: bias dtype %d", what, d->bias_dtype);
    DP_REQUIRE(d->buckets >= 2 && d->buckets <= 64 && (!d->both || d->buckets % 2 == 0) && nb >= 2, "%s: %d buckets",
               what, d->buckets);
    DP_REQUIRE(a->group * d->buckets <= 4096, "%s: %d heads a group x %d buckets", what, a->group, d->buckets);
    a->lse_lo = d->lse_lo;
    a->bias = d->bias; a->bias_f32 = d->bias_dtype == DP_F32; a->buckets = d->buckets; a->both = d->both != 0;
    a->nedge = nb - 1;
    for (int i = 0; i < a->nedge; ++i) {
      a->edge[i] = d->edge[i];
      DP_REQUIRE(a->edge[i] >= (i ? a->edge[i - 1] : 1) && a->edge[i] <= 4096, "%s: bucket edge %d is %d", what, i,
                 a->edge[i]);
    }
  }
  return 0;
}

extern "C" int dp_packed_attn_fwd(const dp_packed_attn* d, void* stream) {
  Args a;
  if (const int rc = dp_packed_attn_args(d, &a, "dp_packed_attn_fwd", false)) return rc;
  if (a.tq == 0) return 0;
  const int64_t need = dp_packed_attn_ws_bytes(d, 0);
  DP_REQUIRE(d->ws_bytes >= need && (d->ws || !need), "dp_packed_attn_fwd: workspace holds %lld bytes, needs %lld",
             (long long)d->ws_bytes, (long long)need);
  const Plan p = plan_of(d);
  DP_REQUIRE((int64_t)p.items * a.hkv <= UINT32_MAX / NT, "dp_packed_attn_fwd: too many tiles");   // a grid's threads
  a.tiles = p.items;
  a.chunk = p.chunk;
  a.splits = p.splits;
  if (p.splits > 1) {
    const int64_t n = (int64_t)a.tq * d->heads;
    a.part = (float*)d->ws;
    a.part_m = a.part + n * p.splits * d->dim;
    a.part_l = a.part_m + n * p.splits;
    a.part_n = (int*)(a.part_l + (d->bias ? n * p.splits : 0));
  }
  hipStream_t s = as_stream(stream);
  const int f = d->fill_tail;
  if (d->dtype == DP_BF16)
    return a.bias ? launch_dim<bf16_t, true>(a, p.wk, f, s) : launch_dim<bf16_t, false>(a, p.wk, f, s);
  return a.bias ? launch_dim<float, true>(a, p.wk, f, s) : launch_dim<float, false>(a, p.wk, f, s);
}
