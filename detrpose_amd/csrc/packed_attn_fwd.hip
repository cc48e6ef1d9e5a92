// Attention over packed sequences, forward (packed_attn.h has the layouts).
//
// One pass over the keys with the running maximum and sum of the softmax: a block owns 128 rows
// (query x head of the group) of one (sequence, key head), 32 a wave, and walks key tiles of BN rows,
// double-buffered in LDS. Per wave and 32 keys: S^T = K Q^T, p = exp(s - m), O^T += V^T P^T; a lane
// holds one row's scores, so the maximum needs one exchange between the wave's halves, and the sum
// none until the end. m moves only when a row's maximum grows by more than 8 in the exponent of 2
// (p stays below 256): the rescaling of O is then rare. p is rounded to bf16 for its product (2^-9
// rms relative, as the output's own rounding); the sum takes it unrounded.
#include "packed_attn.h"
#include <algorithm>

namespace {
using namespace dppa;

constexpr float GROW = 8.f;   // log2 of how far p may pass 1 before m moves

// A row again, key by key: only for a wave whose result holds a NaN. In the products a hidden key's
// weight is 0, but 0 x inf or NaN (a value that causal order hides) is NaN: here hidden keys are not read.
template <typename T, bool BIAS>
__device__ __forceinline__ void slow_row(const Args& a, const Bias& bias, int kvh, int g, int pos, int q0, int k0, int lk,
                                      int lim, int off) {
  const int lane = threadIdx.x & 63;
  const int head = kvh * a.group + g;
  const T* q = (const T*)a.q + (int64_t)(q0 + pos) * a.q_row + head * a.q_head;
  auto score = [&](int j) {
    const T* k = (const T*)a.k + (int64_t)(k0 + j) * a.k_row + kvh * a.k_head;
    float s = 0.f;
    for (int d = 0; d < a.dim; ++d) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
    s *= a.scale;
    if constexpr (BIAS) s += bias.tab[g * bias.nb + bias.bucket(j - pos - off)];
    return s;
  };
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
      const T* v = (const T*)a.v + (int64_t)(k0 + j0 + u) * a.v_row + kvh * a.v_head;
      if (lane < a.dim) o0 = fmaf(w, to_f32(v[lane]), o0);
      if (lane + 64 < a.dim) o1 = fmaf(w, to_f32(v[lane + 64]), o1);
    }
  }
  sum = wave_sum(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* o = (T*)a.out + (int64_t)(q0 + pos) * a.o_row + head * a.o_head;
  if (lane < a.dim) o[lane] = from_f32<T>(o0 * inv);
  if (lane + 64 < a.dim) o[lane + 64] = from_f32<T>(o1 * inv);
}

template <typename T, int DP, int BN, bool BIAS>
__global__ __launch_bounds__(NT, 2) void packed_fwd_kernel(const Args a, int fill_tail) {
  using TL = Tile<T, DP>;
  constexpr int TB = BN * TL::RB, NS = BN / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int kvh = blockIdx.x % a.hkv;
  Item it;
  // the last tiles first: in causal order they have the most keys
  if (!find_item(a.cu_q, a.nseq, a.tq, a.group, BM, fill_tail, a.tiles - 1 - blockIdx.x / a.hkv, it)) return;
  const int q0 = it.start, lq = it.len;
  int k0, lk;
  seq_of(a.cu_k, a.nseq, a.tk, it.b, k0, lk);
  const int off = lk - lq, rows = lq * a.group, row0 = it.tile * BM;
  const int first = row0 + 32 * wave, r = first + (lane & 31);
  const bool ok = r < rows;
  const int rc = min(r, rows - 1), pos = rc / a.group, g = rc - pos * a.group;
  // keys a row sees: [0, lim); of the wave's first and last rows, and of the block's last
  auto limit = [&](int row) {
    return a.causal ? clampi(min(row, rows - 1) / a.group + off + 1, 0, lk) : lk;
  };
  const int lim = limit(r), wmin = limit(first), wmax = first < rows ? limit(first + 31) : 0;
  const int nt = (limit(row0 + BM - 1) + BN - 1) / BN;
  Bias bias{};
  if constexpr (BIAS) bias = bias_setup<T>(a, smem + 4 * TB, kvh);

  u32x4 qf[TL::KS];
  load_frags<T, DP>((const T*)a.q + (int64_t)(q0 + pos) * a.q_row + (kvh * a.group + g) * a.q_head, ok, a.dim, h, qf);

  auto fetch = [&](int j) {
    char* buf = smem + (j & 1) * 2 * TB;
    const int key0 = j * BN, left = lk - key0;
    const i32x4 rk = make_rsrc((const T*)a.k + (int64_t)(k0 + key0) * a.k_row + kvh * a.k_head);
    const i32x4 rv = make_rsrc((const T*)a.v + (int64_t)(k0 + key0) * a.v_row + kvh * a.v_head);
    const int ks = (int)(a.k_row * sizeof(T)), vs = (int)(a.v_row * sizeof(T));
    stage<T, DP, BN>(rk, buf, a.dim, [&](int row) { return row < left ? row * ks : -1; });
    stage<T, DP, BN>(rv, buf + TB, a.dim, [&](int row) { return row < left ? row * vs : -1; });
  };

  // scores in units in which exp(s - m) = exp2((s - m) c): raw products, or, with a bias, scaled ones
  const float c = BIAS ? LOG2E : a.scale * LOG2E;
  float m = -INFINITY, l = 0.f;
  f32x16 o[TL::ND];
#pragma unroll
  for (int t = 0; t < TL::ND; ++t) o[t] = zero16();

  if (nt > 0) fetch(0);
  for (int j = 0; j < nt; ++j) {
    tile_barrier();
    if (j + 1 < nt) fetch(j + 1);
    const char* buf = smem + (j & 1) * 2 * TB;
    const int key0 = j * BN;
    if (key0 >= wmax) continue;
    f32x16 s[NS];
#pragma unroll
    for (int u = 0; u < NS; ++u) s[u] = rows_mma<T, DP>(buf, u, lane, qf);
    if constexpr (BIAS) {
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        const int k32 = key0 + 32 * u, pl = min(first + 31, rows - 1) / a.group + off, pf = first / a.group + off;
        const int one = bias.one_bucket(k32 - pl, k32 + 31 - pf);
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
    if (key0 + BN > wmin) {
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
#pragma unroll
    for (int u = 0; u < NS; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        // with a bias s may be the type's lowest value, whose product with c overflows: subtract first
        s[u][i] = __builtin_amdgcn_exp2f(BIAS ? (s[u][i] - mref) * c : fmaf(s[u][i], c, -mc));
        l += s[u][i];
      }
      cols_mma<T, DP>(buf + TB, u, lane, s[u], o);
    }
  }

  l = half_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bool bad = l != l;
#pragma unroll
  for (int t = 0; t < TL::ND; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      o[t][i] *= inv;
      bad |= o[t][i] != o[t][i];
    }
  if (ok) {
    T* op = (T*)a.out + (int64_t)(q0 + pos) * a.o_row + (kvh * a.group + g) * a.o_head;
#pragma unroll
    for (int t = 0; t < TL::ND; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 32 * t + 8 * e + 4 * h;
        if (d < a.dim) {
          typedef T T4 __attribute__((ext_vector_type(4)));
          T4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = from_f32<T>(o[t][4 * e + i]);
          *reinterpret_cast<T4*>(op + d) = w;
        }
      }
    // for the backward, in the units of its exponent: log2 without, natural with a bias
    if (a.lse && h == 0)
      a.lse[(int64_t)(q0 + pos) * a.hkv * a.group + kvh * a.group + g] =
          l == 0.f ? INFINITY : (BIAS ? m + __logf(l) : m * c + __log2f(l));
  }
  unsigned long long redo = __ballot(bad && ok);
  redo |= redo >> 32;
  for (unsigned left = (unsigned)redo; left; left &= left - 1) {
    const int row = first + __builtin_ctz(left), rp = row / a.group;
    slow_row<T, BIAS>(a, bias, kvh, row - rp * a.group, rp, q0, k0, lk, limit(row), off);
  }
}

template <typename T, int DP, bool BIAS>
int launch(const Args& a, int fill_tail, hipStream_t s) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  const int lds = 4 * BN * Tile<T, DP>::RB + bias_lds(a);
  const auto kern = packed_fwd_kernel<T, DP, BN, BIAS>;
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    DP_REQUIRE(e == hipSuccess, "dp_packed_attn_fwd: %d bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, dim3(a.tiles * a.hkv), dim3(NT), lds, s, a, fill_tail);
  return dp_check_launch("dp_packed_attn_fwd");
}

template <typename T, bool BIAS>
int launch_dim(const Args& a, int fill_tail, hipStream_t s) {
  if (a.dim <= 32) return launch<T, 32, BIAS>(a, fill_tail, s);
  if (a.dim <= 64) return launch<T, 64, BIAS>(a, fill_tail, s);
  return launch<T, 128, BIAS>(a, fill_tail, s);
}

}  // namespace

int dp_packed_attn_args(const dp_packed_attn* d, dppa::Args* a, const char* what, bool backward);

extern "C" int64_t dp_packed_attn_ws_bytes(const dp_packed_attn* d, int32_t backward) {
  if (!d || d->heads <= 0 || d->kv_heads <= 0 || d->tq < 0) return 0;
  if (!backward) return 0;
  const int64_t tiles = (int64_t)d->tq * (d->heads / d->kv_heads) / BM + d->nseq + 1;
  return ((int64_t)d->tq * d->heads + (d->bias ? tiles * d->heads * d->buckets : 0)) * 4;
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
  DP_REQUIRE((d->cu_q && d->cu_k) || d->nseq == 0, "%s: no sequence offsets", what);
  DP_REQUIRE((d->q && d->out) || d->tq == 0, "%s: no queries or output", what);
  DP_REQUIRE((d->k && d->v) || d->tk == 0, "%s: no keys or values", what);
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
  a->q = d->q; a->k = d->k; a->v = d->v; a->out = d->out; a->lse = d->lse;
  a->q_row = d->q_row; a->q_head = d->q_head; a->k_row = d->k_row; a->k_head = d->k_head;
  a->v_row = d->v_row; a->v_head = d->v_head; a->o_row = d->o_row; a->o_head = d->o_head;
  a->cu_q = d->cu_q; a->cu_k = d->cu_k; a->nseq = d->nseq; a->tq = d->tq; a->tk = d->tk;
  a->hkv = d->kv_heads; a->group = d->heads / d->kv_heads; a->dim = d->dim; a->causal = d->causal; a->scale = d->scale;
  const int64_t tiles = (int64_t)d->tq * a->group / BM + d->nseq + 1;
  DP_REQUIRE(tiles * a->hkv < INT32_MAX, "%s: too many tiles", what);
  a->tiles = (int)tiles;
  if (d->bias) {
    const int nb = d->both ? d->buckets / 2 : d->buckets;
    DP_REQUIRE(d->bias_dtype == DP_F32 || d->bias_dtype == d->dtype, "%s: bias dtype %d", what, d->bias_dtype);
    DP_REQUIRE(d->buckets >= 2 && d->buckets <= 64 && (!d->both || d->buckets % 2 == 0) && nb >= 1, "%s: %d buckets",
               what, d->buckets);
    DP_REQUIRE(a->group * d->buckets <= 4096, "%s: %d heads a group x %d buckets", what, a->group, d->buckets);
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
  hipStream_t s = as_stream(stream);
  if (d->dtype == DP_BF16)
    return a.bias ? launch_dim<bf16_t, true>(a, d->fill_tail, s) : launch_dim<bf16_t, false>(a, d->fill_tail, s);
  return a.bias ? launch_dim<float, true>(a, d->fill_tail, s) : launch_dim<float, false>(a, d->fill_tail, s);
}
