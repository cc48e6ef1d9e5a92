// Shared pieces of attention over packed sequences (packed_attn_fwd.hip, packed_attn_bwd.hip).
//
// Rows. The query heads that share a key head are folded into the rows: row r of a (sequence, key
// head) is query r / G, head r % G of the group (G = heads / kv_heads), so one tile of rows reads a key
// tile once for all of them, and the sums over a group's heads in dk / dv are plain row sums.
//
// Matrix layouts (v_mfma_f32_32x32x16_bf16, v_mfma_f32_32x32x2_f32; lane l, h = l >> 5): the A
// operand's row and the B operand's column are l & 31, the accumulator's column is l & 31 and its
// register i holds row 8 (i / 4) + 4 h + i % 4. Every product is arranged so that an accumulator is
// the next product's B operand as it stands: S^T = K Q^T has queries in columns, and the contraction
// of O^T = V^T P^T runs over the accumulator's rows, the slot (h, j) of a 16-row step standing for
// row 16 m + 8 (j / 4) + 4 h + j % 4 on both sides. In bf16 the other side, V^T, is read from the
// row-major tile with the transposing LDS read (4 rows x 16 columns per 16 lanes), in f32 with one
// 4-byte read per step.
//
// Tiles. Rows of DP elements (dim padded to 32, 64 or 128; the padding reads as zero), filled by
// direct HBM -> LDS loads whose buffer descriptor returns zero for rows outside the sequence: what
// lies there (another sequence, an unwritten cache row) never enters a product. A row's 16-byte chunks
// are permuted by its number (Tile::swz); the permutation is applied to the global address, because
// the LDS side of such a load is contiguous per wave.
#pragma once
#include "common.h"
#include "conv_lds.h"

namespace dppa {

using dpconv::i32x4;
using dpconv::make_rsrc;
using dpconv::OOB;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float LN2 = 0.69314718055994530942f;
constexpr int NT = 256;     // threads of a block: 4 waves, 32 rows (or keys) each
constexpr int BM = 128;     // rows (keys, in the dk / dv kernel) of a block

// dk / dv: a run [w0, w1) of a key tile's walk over the queries; row: where its part goes, if there are several
struct alignas(16) Piece { int start, len, start2, len2, tile, w0, w1, parts, begins, row, unused[2]; };

// what a kernel needs to know; strides in elements
struct Args {
  const void *q, *k, *v;
  void* out;
  float *lse, *lse_lo;
  bf16_t* out_lo;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
  const int32_t *cu_q, *cu_k;
  int nseq, tq, tk, hkv, group, dim, causal, tiles;
  float scale;
  // split keys (forward): key chunk at least, most chunks of one sequence, and where the parts go
  int chunk, splits;
  float *part, *part_m, *part_l;
  int* part_n;
  // bias
  const void* bias;
  int bias_f32, buckets, both, nedge;
  int32_t edge[64];
  // backward
  const void* dout;
  int64_t g_row, g_head;
  void *dq, *dk, *dv;
  float* dsum;
  float* dbias_part;
  // dk / dv, of one key head: blocks, units of a share at least, places for parts, shares and pieces at most
  int kblocks, kunits, kslots, kshares, kpieces;
  float* kv_part;
  int2 *kv_n, *kv_share;
  Piece* kv_piece;
};

// A wave-uniform value in a scalar register (the empty asm keeps it there: the compiler drops a
// readfirstlane of what it knows to be uniform and may then carry on with vector instructions)
__device__ __forceinline__ int uniform(int x) {
  x = __builtin_amdgcn_readfirstlane(x);
  asm("" : "+s"(x));
  return x;
}

// 16 bytes a lane from rsrc + off (zero outside) to LDS, lane L at at + 16 L; 4 bytes a lane for the first n
// lanes. A FRESH descriptor may just have been written by vector instructions (readfirstlane), which a memory
// instruction may read 5 wait states later, and m0 one after its write: the nop counts these, as the
// compiler does not look into the asm. Completion is waited for by hand.
template <bool FRESH = true>
__device__ __forceinline__ void dma16(const i32x4& rsrc, const char* at, int off, int soff = 0) {
  const unsigned m0 = __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>(at));
  i32x4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w) r[w] = __builtin_amdgcn_readfirstlane(rsrc[w]);
  if (FRESH)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0), "v"(off), "s"(r),
                 "s"(soff)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0), "v"(off), "s"(r),
                 "s"(soff)
                 : "memory");
}
__device__ __forceinline__ void dma4(const i32x4& rsrc, const char* at, int off, int n) {
  const unsigned m0 = __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>(at));
  i32x4 r;
#pragma unroll
  for (int w = 0; w < 4; ++w) r[w] = __builtin_amdgcn_readfirstlane(rsrc[w]);
  if ((int)(threadIdx.x & 63) < n)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(m0), "v"(off), "s"(r)
                 : "memory");
}

template <typename T> struct Tr;
template <> struct Tr<bf16_t> { static constexpr int VN = 8; };
template <> struct Tr<float> { static constexpr int VN = 4; };

template <typename T, int DP>
struct Tile {
  static constexpr int VN = Tr<T>::VN;          // elements of a 16-byte chunk
  static constexpr int CPR = DP / VN;           // chunks of a row
  static constexpr int RB = DP * (int)sizeof(T);
  static constexpr int KS = CPR / 2;            // chunk pairs: the steps of a product over dim
  static constexpr int ND = DP / 32;            // 32-wide column tiles
  // A tile lies in groups of 1 KB (what one wave's load writes) GS bytes apart, and a row's chunks are
  // permuted by swz, so that over the 16 slots of 16 bytes that one LDS cycle serves, the equal chunks of 16
  // rows (products over dim) and what one column read takes at once (bf16: 64 bytes of each of 4
  // rows; f32: 128 bytes of rows r and r + 4) lie on different slots. The groups' spacing takes part of
  // that from the permutation, which leaves few different addresses to keep in registers.
  static constexpr int RG = 1024 / RB, GS = 1040;
  static constexpr int PERIOD = sizeof(T) == 2 || CPR == 8 ? RG : 8;   // of swz, in rows
  __device__ static __forceinline__ int swz(int row) {
    if (sizeof(T) == 2) return CPR == 16 ? (row & 3) << 2 : CPR == 8 ? ((row & 2) << 1) | ((row & 4) >> 1) : (row >> 2) & 3;
    if (CPR == 32) return ((row ^ (row >> 2)) & 1) << 3;
    return CPR == 16 ? ((row & 3) << 2) ^ ((row & 4) << 1) : ((row & 2) << 1) | ((row & 4) >> 1);
  }
  __device__ static __forceinline__ int off(int row) { return row / RG * GS + row % RG * RB; }
  static constexpr int bytes(int rows) { return rows / RG * GS; }
};

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// one chunk-pair step of a product over dim: 16 elements in bf16, 8 in f32
template <typename T>
__device__ __forceinline__ f32x16 mma_step(const u32x4& a, const u32x4& b, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
    return c;
  }
}

// a lane's operands for products over dim: its chunk of step s of row 32 u + (l & 31). swz leaves the low
// bit (and with 16 chunks a row the low two) of a chunk alone, so the steps share few addresses
template <typename T, int DP>
struct RowReader {
  using TL = Tile<T, DP>;
  static constexpr int SH = sizeof(T) == 2 && TL::CPR == 16 ? 2 : sizeof(T) == 2 && TL::CPR == 4 ? 0 : 1;
  const char* base;
  int f, h;
  __device__ __forceinline__ RowReader(const char* tile, int lane)
      : base(tile + TL::off(lane & 31) + (SH ? (lane >> 5) * 16 : 0)), f(TL::swz(lane & 31)), h(SH ? 0 : lane >> 5) {}
  __device__ __forceinline__ bf16x8 read(int u, int s) const {
    const int c = 2 * s + h, lo = c & ((1 << SH) - 1);
    return *reinterpret_cast<const bf16x8*>(base + TL::bytes(32) * u + lo * 16 + (((c - lo) ^ f) << 4));
  }
};

// bf16: columns 32 t + (l & 31) of rows 32 u + 16 m + (the step's slots), transposed by the read
template <int DP>
struct ColReader {
  using TL = Tile<bf16_t, DP>;
  // the second four rows of a step are 8 further on
  static constexpr int D8 = TL::RG <= 8 ? 8 / TL::RG * TL::GS : 8 * TL::RB, D16 = 16 / TL::RG * TL::GS;
  static constexpr bool WHOLE = TL::CPR == 16;   // swz permutes whole column tiles
  const char* base;
  int f, f8, c;
  __device__ __forceinline__ ColReader(const char* tile, int lane) {
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2), p4 = lane & 3;   // r: row % 8 of every row read
    c = 2 * ((lane >> 4) & 1) + (p4 >> 1);
    base = tile + TL::off(r) + (p4 & 1) * 8 + (WHOLE ? c * 16 : 0);
    f = TL::swz(r);
    f8 = TL::RG <= 8 ? f : TL::swz(r + 8);
    if (WHOLE) c = 0;
  }
  __device__ __forceinline__ bf16x8 read(int u, int m, int t) const {
    const char* at = base + TL::bytes(32) * u + m * D16;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(at + (((4 * t + c) ^ f) << 4)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(at + D8 + (((4 * t + c) ^ f8) << 4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
};

// c[u] = rows 32 (sub + u) ... of the tile x the lane's column fragments, the N chains side by side
template <typename T, int DP, int N>
__device__ __forceinline__ void rows_mma_n(const char* tile, int sub, int lane, const u32x4 (&b)[Tile<T, DP>::KS],
                                           f32x16 (&c)[N]) {
  using TL = Tile<T, DP>;
  const RowReader<T, DP> rd(tile + TL::bytes(32) * sub, lane);
#pragma unroll
  for (int u = 0; u < N; ++u) c[u] = zero16();
#pragma unroll
  for (int s = 0; s < TL::KS; ++s)
#pragma unroll
    for (int u = 0; u < N; ++u) c[u] = mma_step<T>(__builtin_bit_cast(u32x4, rd.read(u, s)), b[s], c[u]);
}
template <typename T, int DP>
__device__ __forceinline__ f32x16 rows_mma(const char* tile, int sub, int lane, const u32x4 (&b)[Tile<T, DP>::KS]) {
  f32x16 c[1];
  rows_mma_n<T, DP, 1>(tile, sub, lane, b, c);
  return c[0];
}

// the bf16 column operand of two 16-row steps from an accumulator
__device__ __forceinline__ void pack_p(const f32x16& p, bf16x8 (&b)[2]) {
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int j = 0; j < 8; ++j) b[m][j] = (bf16_t)p[8 * m + j];
}

// acc[t] += tile^T (columns 32 t ...) x p, contracted over the tile's rows 32 sub .. 32 sub + 31
template <int DP>
__device__ __forceinline__ void cols_mma_packed(const char* tile, int sub, int lane, const bf16x8 (&p)[2],
                                                f32x16 (&acc)[Tile<bf16_t, DP>::ND]) {
  const ColReader<DP> rd(tile, lane);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < Tile<bf16_t, DP>::ND; ++t)
      acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rd.read(sub, m, t), p[m], acc[t], 0, 0, 0);
}

template <typename T, int DP>
__device__ __forceinline__ void cols_mma(const char* tile, int sub, int lane, const f32x16& p,
                                         f32x16 (&acc)[Tile<T, DP>::ND]) {
  using TL = Tile<T, DP>;
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    bf16x8 b[2];
    pack_p(p, b);
    cols_mma_packed<DP>(tile, sub, lane, b, acc);
  } else {
    const int c = (lane & 31) >> 2, w = (lane & 3) * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = 8 * (i / 4) + 4 * h + (i & 3);
      const char* base = tile + TL::bytes(32) * sub + TL::off(row) + w;
      const int f = TL::swz(row);
#pragma unroll
      for (int t = 0; t < TL::ND; ++t) {
        const float a = *reinterpret_cast<const float*>(base + (((8 * t + c) ^ f) << 4));
        acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[i], acc[t], 0, 0, 0);
      }
    }
  }
}

// ROWS rows, stride bytes apart, of which the first `valid` exist: one lane offset serves every pass (the
// rows of two passes are a whole period of swz apart, so a chunk's place is the same). A whole tile's
// passes share a descriptor and differ in the scalar offset; the last, partial one moves the descriptor's
// base instead, whose length ends with the last row (a scalar offset past the length would wrap the
// hardware's range check). lane_off(): that offset.
template <typename T, int DP, int THREADS = NT>
__device__ __forceinline__ int lane_off(int stride, int dim) {
  using TL = Tile<T, DP>;
  static_assert(THREADS / TL::CPR % TL::PERIOD == 0, "whole periods of swz a pass");
  const int t = THREADS == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int row = t / TL::CPR, c = (t % TL::CPR) ^ TL::swz(row);
  return c * TL::VN < dim ? row * stride + c * 16 : OOB;
}
template <typename T, int DP, int ROWS, int THREADS = NT>
__device__ __forceinline__ void stage_rows(const T* base, int stride, int valid, char* tile, int dim, int off,
                                           int wave) {
  using TL = Tile<T, DP>;
  constexpr int RPP = THREADS / TL::CPR;   // rows of a pass
  static_assert(ROWS % RPP == 0, "whole passes");
  if (valid >= ROWS) {
    const i32x4 r = make_rsrc(base);
    dma16(r, tile + wave * TL::GS, off);
#pragma unroll
    for (int it = 1; it < ROWS / RPP; ++it)
      dma16<false>(r, tile + (it * (THREADS / 64) + wave) * TL::GS, off, it * RPP * stride);
    return;
  }
  const int end = (valid - 1) * stride + dim * (int)sizeof(T);   // below 2^31: stride < 2^24
#pragma unroll
  for (int it = 0; it < ROWS / RPP; ++it) {
    i32x4 r = make_rsrc(reinterpret_cast<const char*>(base) + (int64_t)it * RPP * stride);
    r[2] = max(end - it * RPP * stride, 0);
    dma16(r, tile + (it * (THREADS / 64) + wave) * TL::GS, off);
  }
}

// the lane's fragments of one global row as a B operand (zero when !ok and past dim)
template <typename T, int DP>
__device__ __forceinline__ void load_frags(const T* row, bool ok, int dim, int h, u32x4 (&f)[Tile<T, DP>::KS]) {
#pragma unroll
  for (int s = 0; s < Tile<T, DP>::KS; ++s) {
    const int e = (2 * s + h) * Tr<T>::VN;
    f[s] = ok && e < dim ? *reinterpret_cast<const u32x4*>(row + e) : u32x4{0, 0, 0, 0};
  }
}

// both halves of the wave get a (op) b of lanes l and l ^ 32
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// everything issued to LDS so far has landed, for every wave of the block
__device__ __forceinline__ void tile_barrier() {
  dpconv::wait_vmcnt<0>();
  __syncthreads();
}

// four results of a row: rounded, and in bf16, where the backward wants it, what the rounding left off
template <typename T>
__device__ __forceinline__ void put4(T* out, bf16_t* lo, const f32x4& x) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = from_f32<T>(x[e]);
  *reinterpret_cast<T4*>(out) = w;
  if constexpr (sizeof(T) == 2) {
    if (lo) {
      bf16x4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (bf16_t)(x[e] - (float)w[e]);
      *reinterpret_cast<bf16x4*>(lo) = r;
    }
  }
}

// The log of a row's softmax denominator, l times the exponential of m, in the backward's units: log2 without a
// bias, natural with one. A learned bias can be far larger than the scores' differences (a mask of -1e9, the type's
// lowest value): m + log l then rounds log l away and the backward's weights would not add up to 1, so with a bias
// lse_lo takes what the sum's rounding left off, in log2.
template <bool BIAS>
__device__ __forceinline__ void put_lse(const Args& a, int64_t at, float m, float l) {
  if (!a.lse) return;
  if constexpr (BIAS) {
    const float g = __logf(l), x = m + g, y = x - m;
    a.lse[at] = l == 0.f ? INFINITY : x;
    if (a.lse_lo) a.lse_lo[at] = l == 0.f ? 0.f : ((m - (x - y)) + (g - y)) * LOG2E;
  } else {
    a.lse[at] = l == 0.f ? INFINITY : m + __log2f(l);
  }
}

// ---------------------------------------------------------------- which sequence a block works on
// The lengths are on the device only: a launch has as many blocks as the packed total allows at
// most, and every wave finds its block's (sequence, tile) by a scan over the sequences, 64 at a time.
// nseq counts one more when the rows behind the last sequence are an item of their own (tail).
struct Item { int b, sub, start, len, start2, len2; };   // start2, len2: of the other side's rows

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// cu's sequences, a sequence counting items(its length, its length by cu2) blocks, each of which walks that second
// length; it.sub: which of them idx is. Of up to 64 sequences those with longer walks come later (blocks are
// handed out from the last idx on, so that the longest start first: a 4096-key prompt in front of
// shorter ones 225 -> 214 us); more stay in order.
template <typename COUNT>
__device__ __forceinline__ bool search_item(const int32_t* cu, int total, const int32_t* cu2, int total2, int nseq,
                                            bool tail, int idx, COUNT items, Item& it) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  const int n = nseq + (tail ? 1 : 0);
  for (int base = 0; base < n; base += 64) {
    const int b = base + lane;
    int start = 0, len = 0, start2 = 0, walk = 0;
    if (b < n) {
      // all four at once: a small call's time is the number of round trips
      const int c0 = cu[min(b, nseq)], c1 = cu[min(b + 1, nseq)], d0 = cu2[min(b, nseq)], d1 = cu2[min(b + 1, nseq)];
      start = b ? clampi(c0, 0, total) : 0;
      len = max(0, (b < nseq ? clampi(c1, 0, total) : total) - start);
      start2 = b && b < nseq ? clampi(d0, 0, total2) : 0;
      walk = b < nseq ? max(0, clampi(d1, 0, total2) - start2) : 0;
    }
    const int cnt = len ? items(len, walk) : 0;
    int from = 0, all = 0;   // items in front of this lane's, and of all lanes
    if (n <= 64) {
      for (int o = 0; o < n; ++o) {
        const int ow = __builtin_amdgcn_readlane(walk, o), oc = __builtin_amdgcn_readlane(cnt, o);
        from += ow < walk || (ow == walk && o < lane) ? oc : 0;
        all += oc;
      }
    } else {
      int inc = cnt;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
      }
      from = inc - cnt;
      all = __shfl(inc, 63, 64);
    }
    if (idx < before + all) {
      const unsigned long long m = __ballot(idx - before >= from && idx - before < from + cnt);
      const int l = __ffsll((long long)m) - 1;
      it.b = base + l;
      it.sub = idx - before - __shfl(from, l, 64);
      it.start = __shfl(start, l, 64);
      it.len = __shfl(len, l, 64);
      it.start2 = __shfl(start2, l, 64);
      it.len2 = __shfl(walk, l, 64);
      return true;
    }
    before += all;
  }
  return false;
}

template <typename COUNT>
__device__ __forceinline__ bool find_item(const int32_t* cu, int total, const int32_t* cu2, int total2, int nseq,
                                          bool tail, int idx, COUNT items, Item& it) {
  Item x{};
  const bool found = search_item(cu, total, cu2, total2, nseq, tail, idx, items, x);
  // made scalar here, behind the search's loop, whose exit the compiler takes for one that lanes leave singly
  it = Item{uniform(x.b), uniform(x.sub), uniform(x.start), uniform(x.len), uniform(x.start2), uniform(x.len2)};
  return uniform(found) != 0;
}

// start and length of sequence b (nothing for the tail)
__device__ __forceinline__ int2 seq_at(const int32_t* cu, int nseq, int total, int b) {
  const int start = b && b < nseq ? clampi(cu[b], 0, total) : 0;
  return int2{start, b < nseq ? max(0, clampi(cu[b + 1], 0, total) - start) : 0};
}
// ---------------------------------------------------------------- relative position bias
// LDS: tab[g][bucket] f32 of the group's heads, then lut[n] = bucket of distance n, n <= last (the
// distance from which on every one is in the last bucket).
struct Bias {
  const float* tab;
  const uint8_t* lut;
  int nb, last, half, both;
  __device__ __forceinline__ int bucket(int rel) const {
    const int n = min(both ? abs(rel) : max(-rel, 0), last);
    return lut[n] + (rel > 0 ? half : 0);
  }
  // the bucket that every distance in [lo, hi] falls into, or -1 (there may be several)
  __device__ __forceinline__ int one_bucket(int lo, int hi) const {
    if (hi <= -last) return lut[last];
    if (both ? lo >= last : lo >= 0) return both ? lut[last] + half : 0;
    return -1;
  }
};

static inline int bias_lds(const Args& a) {
  return a.bias ? a.group * a.buckets * 4 + ((a.nedge ? a.edge[a.nedge - 1] : 0) + 1 + 15) / 16 * 16 : 0;
}

template <typename T, int THREADS = NT>
__device__ __forceinline__ Bias bias_setup(const Args& a, char* lds, int kvh) {
  float* tab = reinterpret_cast<float*>(lds);
  uint8_t* lut = reinterpret_cast<uint8_t*>(tab + a.group * a.buckets);
  const int heads = a.hkv * a.group;
  for (int i = threadIdx.x; i < a.group * a.buckets; i += THREADS) {
    const int g = i / a.buckets, b = i - g * a.buckets;
    const int64_t at = (int64_t)b * heads + kvh * a.group + g;
    tab[i] = a.bias_f32 ? reinterpret_cast<const float*>(a.bias)[at] : to_f32(reinterpret_cast<const T*>(a.bias)[at]);
  }
  const int last = a.nedge ? a.edge[a.nedge - 1] : 0;
  for (int n = threadIdx.x; n <= last; n += THREADS) {
    int b = 0;
    for (int e = 0; e < a.nedge; ++e) b += a.edge[e] <= n;
    lut[n] = (uint8_t)b;
  }
  __syncthreads();
  return Bias{tab, lut, a.buckets, last, a.both ? a.buckets / 2 : 0, a.both};
}

}  // namespace dppa
