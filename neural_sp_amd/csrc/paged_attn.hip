// paged_attn.hip -- attention of a few new tokens over a long row of keys: a paged key / value cache (decoding: self
// attention over the prefix) or a plain [B, T, heads, d] tensor (decoding: source attention over the encoder's states), and
// the append to such a cache.
//
//   out[b, t, h, :] = sum_j p_j v_j,  p = softmax_j(scale q[b, t, h, :] . k_j),  j < len[b]
//
// Every key and value is read once: 2 len d bytes-per-element against 4 len d flops per query row, so HBM bounds the call
// and, for short rows, the launch and the latency of two dependent loads (page number, then key).
//
// One workgroup takes up to 16 query rows that share a key head (query heads of the group x new tokens) and one stretch of
// the keys; its four waves take 32-key tiles in turn, each with its own running maximum and sum, and meet once at the end
// in LDS.  A row's keys are split over several workgroups when there are few rows; a second small kernel joins the parts.
// Scores are S^T = K Q^T with the query on the lane's column, so maximum, sum and rescaling are per lane and the
// probabilities already are the operand of O^T = V^T P^T.  Keys and values go from memory into the operands' registers, the
// next tile's while this one is worked on; a value operand wants eight KEYS of one dimension per lane where memory has
// dimensions side by side, so a lane loads d / 16 dimensions of its eight keys and transposes 8 x d / 16 in registers.
// Probabilities enter the product as bf16 high + low parts (16 bits): the matrix cores are idle enough that the second
// product is free, and the result's only rounding to bf16 is the last one.  Both parts are positive where the probability is, so
// that an infinite value stays one: the high part is cut off below the probability, and a low part of zero is 2^-24 of it.
//
// Scores of -inf alone have no softmax.  Over states the result is NaN, as the training kernel and the definition have it; over
// a cache such a row is one whose keys are all absent: zeros.
#include "attn_frag.h"
#include <algorithm>

namespace {

struct DecodeArgs {
  const void* q;
  void* out;
  const void* k;
  const void* v;
  const int* table;
  const int* lens;
  const void* k_new;
  const void* v_new;
  float* ws;
  int B, H, Hkv, D, Tq, page, width, nsplit, chunk, cap, rows, ngrp;
  unsigned page_magic, n_pages;
  long long q_sb, q_st, q_sh, k_sp, k_ss, k_sh, v_sp, v_ss, v_sh, kn_sb, kn_sh, vn_sb, vn_sh;
  float sl2;
};

// j / page for any page size: one multiply-high, its estimate is the quotient or one less
__device__ __forceinline__ void page_split(const DecodeArgs& p, unsigned j, unsigned& pg, unsigned& slot) {
  pg = (unsigned)(((unsigned long long)j * p.page_magic) >> 32);
  slot = j - pg * (unsigned)p.page;
  if (slot >= (unsigned)p.page) { ++pg; slot -= (unsigned)p.page; }
}

// is there such a page (a negative number is behind every page)
__device__ __forceinline__ bool page_there(const DecodeArgs& p, int id) { return (unsigned)id < p.n_pages; }

// VW consecutive elements of a value row
template <typename T, int VW>
struct ValueRow;
template <int VW>
struct ValueRow<float, VW> {
  float x[VW];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (VW == 2) {
      const float2 a = *reinterpret_cast<const float2*>(p);
      x[0] = a.x; x[1] = a.y;
    } else {
#pragma unroll
      for (int i = 0; i < VW / 4; ++i) {
        const f32x4 a = reinterpret_cast<const f32x4*>(p)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = a[e];
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < VW; ++i) x[i] = 0.f;
  }
};
template <int VW>
struct ValueRow<__bf16, VW> {
  unsigned x[VW / 2];
  __device__ __forceinline__ void load(const __bf16* p) {
    if constexpr (VW == 2) {
      x[0] = *reinterpret_cast<const unsigned*>(p);
    } else if constexpr (VW == 4) {
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      x[0] = a.x; x[1] = a.y;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < VW / 2; ++i) x[i] = 0u;
  }
};

// o[j] (rows: dimension m * VW + j, column: query) += sum over the tile's 32 keys; v[4 kf + e] = key 16 kf + 4 g + e
template <int VW>
__device__ __forceinline__ void value_product(f32x4 (&o)[VW], const ValueRow<float, VW> (&v)[8], const float (&pr)[2][4]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < VW; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i].x[j], pr[i >> 2][i & 3], o[j], 0, 0, 0);
}
template <int VW>
__device__ __forceinline__ void value_product(f32x4 (&o)[VW], const ValueRow<__bf16, VW> (&v)[8], const float (&pr)[2][4]) {
  bf16x8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = pr[i >> 2][i & 3], h = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
    hi[i] = (__bf16)h;
    lo[i] = (__bf16)fmaxf(x - h, x * 5.9604644775390625e-8f);
  }
#pragma unroll
  for (int w = 0; w < VW / 2; ++w) {
    nsp_u32x4 even, odd;   // dimensions 2 w and 2 w + 1 of the eight keys
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      even[i] = (v[2 * i].x[w] & 0xFFFFu) | (v[2 * i + 1].x[w] << 16);
      odd[i] = (v[2 * i].x[w] >> 16) | (v[2 * i + 1].x[w] & 0xFFFF0000u);
    }
    const bf16x8 a = __builtin_bit_cast(bf16x8, even), c = __builtin_bit_cast(bf16x8, odd);
    o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, hi, o[2 * w], 0, 0, 0);
    o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c, hi, o[2 * w + 1], 0, 0, 0);
    o[2 * w] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, lo, o[2 * w], 0, 0, 0);
    o[2 * w + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c, lo, o[2 * w + 1], 0, 0, 0);
  }
}

// where the keys are: CONTIG = one [T, heads, d] stretch per sequence; BLOCK16 = pages of a multiple of 16 keys, so the page
// of a 16-key block is uniform over the wave (scalar loads); ROWS = any page size, looked up row by row
enum { CONTIG = 0, BLOCK16 = 1, ROWS = 2 };

template <typename T, int DP>
struct Tile {
  static constexpr int NS = DP / (4 * AttnElem<T>::CE), VW = DP / 16;
  typename AttnElem<T>::chunk k[2][NS];
  ValueRow<T, VW> v[8];
  unsigned ok;   // BLOCK16: bit kf; ROWS: bit 4 kf + e of the lane's eight keys
};

// BLOCK16: pages and slots of a tile's two 16-key blocks.  Looked up ahead of the keys, and without regard to the sequence's
// length, so that the first tile's lookup runs beside the load of that length and the others' behind the tile before.
struct TilePages {
  int id[2], slot[2];
};
template <int MODE>
__device__ __forceinline__ TilePages load_pages(const DecodeArgs& p, const int* tab, int j0) {
  TilePages t;
  if constexpr (MODE == BLOCK16) {
#pragma unroll
    for (int kf = 0; kf < 2; ++kf) {
      unsigned pg, slot;
      page_split(p, (unsigned)min(j0 + 16 * kf, p.cap - 16), pg, slot);       // (cap: a multiple of the page)
      t.id[kf] = tab[pg];
      t.slot[kf] = (int)slot;
    }
  }
  return t;
}

template <typename T, int DP, int MODE>
__device__ __forceinline__ void load_tile(Tile<T, DP>& t, const DecodeArgs& p, const T* kb, const T* vb, const int* tab,
                                          const TilePages& pages, int j0, int end, int r, int g, bool full_d) {
  typedef AttnElem<T> E;
  constexpr int NS = Tile<T, DP>::NS, VW = Tile<T, DP>::VW;
  t.ok = 0u;
  const bool v_in = full_d || r * VW < p.D;
#pragma unroll
  for (int kf = 0; kf < 2; ++kf) {
    const int jb = j0 + 16 * kf;
    const T* krow;
    const T* vrow[4];
    bool kok = true, vok[4] = {true, true, true, true};
    if constexpr (MODE == CONTIG) {
      krow = kb + (long long)min(jb + r, end - 1) * p.k_ss;
#pragma unroll
      for (int e = 0; e < 4; ++e) vrow[e] = vb + (long long)min(jb + 4 * g + e, end - 1) * p.v_ss;
    } else if constexpr (MODE == BLOCK16) {
      kok = jb < end && page_there(p, pages.id[kf]);
      const long long at = kok ? pages.id[kf] : 0;
      const int slot = kok ? pages.slot[kf] : 0, top = kok ? min(15, end - 1 - jb) : 0;
      krow = kb + at * p.k_sp + (long long)(slot + min(r, top)) * p.k_ss;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vrow[e] = vb + at * p.v_sp + (long long)(slot + min(4 * g + e, top)) * p.v_ss;
        vok[e] = kok;
      }
      t.ok |= kok ? (1u << kf) : 0u;
    } else {
      unsigned pg, slot;
      page_split(p, (unsigned)min(jb + r, end - 1), pg, slot);
      int id = tab[pg];
      kok = page_there(p, id);
      krow = kb + (long long)(kok ? id : 0) * p.k_sp + (long long)slot * p.k_ss;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        page_split(p, (unsigned)min(jb + 4 * g + e, end - 1), pg, slot);
        id = tab[pg];
        vok[e] = page_there(p, id);
        vrow[e] = vb + (long long)(vok[e] ? id : 0) * p.v_sp + (long long)slot * p.v_ss;
        t.ok |= vok[e] ? (1u << (4 * kf + e)) : 0u;
      }
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = (4 * s + g) * E::CE;
      if (kok && (full_d || c < p.D)) t.k[kf][s] = *reinterpret_cast<const typename E::chunk*>(krow + c);
      else t.k[kf][s] = E::zero();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (vok[e] && v_in) t.v[4 * kf + e].load(vrow[e] + r * VW);
      else t.v[4 * kf + e].clear();      // a page that is not there: its probability is 0, 0 x stale memory may not be
    }
  }
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__(256) void decode_attn_kernel(const DecodeArgs p) {
  typedef AttnElem<T> E;
  constexpr int NS = Tile<T, DP>::NS, VW = Tile<T, DP>::VW;
  constexpr int LP = DP + 4;
  __shared__ __attribute__((aligned(16))) float part_o[4][16][LP];
  __shared__ float part_m[4][16], part_l[4][16], new_s[16];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int split = blockIdx.x, b = blockIdx.z;
  const int hkv = (int)blockIdx.y / p.ngrp, grp = (int)blockIdx.y % p.ngrp;
  const int G = p.H / p.Hkv, row0 = grp * 16, nrow = min(16, p.rows - row0);
  const int* tab = MODE == CONTIG ? nullptr : p.table + (long long)b * p.width;
  const int start = split * p.chunk;
  int j0 = start + 32 * wave;
  TilePages pages = load_pages<MODE>(p, tab, j0);
  int len = p.lens ? p.lens[b] : p.cap;
  const bool unused = MODE != CONTIG && len < 0;
  len = max(0, min(len, p.cap));
  // an utterance without a visible key: the finite mask value of the training path makes its softmax uniform over ALL keys
  const bool uniform = MODE == CONTIG && len == 0;
  if (uniform) len = p.cap;
  const int end = min(len, start + p.chunk);
  if (split > 0 && start >= len) return;
  const bool full_d = p.D == DP;
  const T* kb = reinterpret_cast<const T*>(p.k) + (long long)hkv * p.k_sh;
  const T* vb = reinterpret_cast<const T*>(p.v) + (long long)hkv * p.v_sh;
  if constexpr (MODE == CONTIG) {
    kb += (long long)b * p.k_sp;
    vb += (long long)b * p.v_sp;
  }
  const T* qb = reinterpret_cast<const T*>(p.q) + (long long)b * p.q_sb;

  // this lane's query column
  typename E::chunk qf[NS];
  {
    const int rr = row0 + min(r, nrow - 1);
    const T* qr = qb + (long long)(rr / G) * p.q_st + (long long)(hkv * G + rr % G) * p.q_sh;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = (4 * s + g) * E::CE;
      qf[s] = full_d || c < p.D ? *reinterpret_cast<const typename E::chunk*>(qr + c) : E::zero();
    }
  }
  f32x4 o[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  Tile<T, DP> cur, nxt;
  if (j0 < end) {
    load_tile<T, DP, MODE>(cur, p, kb, vb, tab, pages, j0, end, r, g, full_d);
    pages = load_pages<MODE>(p, tab, j0 + 128);
  }
  while (j0 < end) {
    const int jn = j0 + 128;
    if (jn < end) {
      load_tile<T, DP, MODE>(nxt, p, kb, vb, tab, pages, jn, end, r, g, full_d);
      pages = load_pages<MODE>(p, tab, jn + 128);
    }
    float pr[2][4];
    float mx = -INFINITY;
#pragma unroll
    for (int kf = 0; kf < 2; ++kf) {
      f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i) s = E::mma(cur.k[kf][i], qf[i], s);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool seen = j0 + 16 * kf + 4 * g + e < end &&
                          (MODE == CONTIG || ((cur.ok >> (MODE == BLOCK16 ? kf : 4 * kf + e)) & 1u));
        const float x = uniform ? 0.f : s[e] * p.sl2;
        pr[kf][e] = seen ? x : -INFINITY;
        mx = attn_max(mx, pr[kf][e]);
      }
    }
    const float mn = attn_max(m, attn_max4(mx));
    const float base = mn == -INFINITY ? 0.f : mn;     // (nothing seen so far: every exponent below is -inf)
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int kf = 0; kf < 2; ++kf)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[kf][e] = __builtin_amdgcn_exp2f(pr[kf][e] - base);
        l += pr[kf][e];
      }
#pragma unroll
    for (int j = 0; j < VW; ++j) o[j] *= alpha;
    if (j0 + 32 > end) {      // what was loaded for keys behind the end: 0 x an infinite last value would be NaN
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + 16 * (i >> 2) + 4 * g + (i & 3) >= end) cur.v[i].clear();
    }
    value_product<VW>(o, cur.v, pr);
    cur = nxt;
    j0 = jn;
  }
  l = attn_sum4(l);

  // the new token's own key and value: stored to the cache by one workgroup, and one more part of the join
  bool has_new = false;
  if (MODE != CONTIG && p.k_new != nullptr && split == 0 && !unused && len < p.cap) {
    unsigned pg, slot;
    page_split(p, (unsigned)len, pg, slot);
    const int id = tab[pg];
    if (page_there(p, id)) {
      has_new = true;
      const T* kn = reinterpret_cast<const T*>(p.k_new) + (long long)b * p.kn_sb + (long long)hkv * p.kn_sh;
      const T* vn = reinterpret_cast<const T*>(p.v_new) + (long long)b * p.vn_sb + (long long)hkv * p.vn_sh;
      if (grp == 0 && (int)threadIdx.x < p.D) {
        T* kd = const_cast<T*>(kb) + (long long)id * p.k_sp + (long long)slot * p.k_ss;
        T* vd = const_cast<T*>(vb) + (long long)id * p.v_sp + (long long)slot * p.v_ss;
        kd[threadIdx.x] = kn[threadIdx.x];
        vd[threadIdx.x] = vn[threadIdx.x];
      }
      for (int q = wave; q < nrow; q += 4) {
        const int rr = row0 + q;
        const T* qr = qb + (long long)(rr / G) * p.q_st + (long long)(hkv * G + rr % G) * p.q_sh;
        float s = 0.f;
        for (int d = lane; d < p.D; d += 64) s = fmaf(E::to_f32(qr[d]), E::to_f32(kn[d]), s);
        s = wave_reduce_sum(s);
        if (lane == 0) new_s[q] = s * p.sl2;
      }
    }
  }

  if (g == 0) { part_m[wave][r] = m; part_l[wave][r] = l; }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int j = 0; j < VW; ++j) part_o[wave][r][(4 * g + e) * VW + j] = o[j][e];
  __syncthreads();
  const int q = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * VW;
  if (q >= nrow) return;
  float M = has_new ? new_s[q] : -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) M = attn_max(M, part_m[w][q]);
  const float base = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) acc[j] = 0.f;
  if (has_new) {
    const float f = __builtin_amdgcn_exp2f(new_s[q] - base);
    const T* vn = reinterpret_cast<const T*>(p.v_new) + (long long)b * p.vn_sb + (long long)hkv * p.vn_sh;
    L = f;
#pragma unroll
    for (int j = 0; j < VW; ++j) acc[j] = d0 + j < p.D ? f * E::to_f32(vn[d0 + j]) : 0.f;
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(part_m[w][q] - base);
    L = fmaf(f, part_l[w][q], L);
#pragma unroll
    for (int j = 0; j < VW; ++j) acc[j] = fmaf(f, part_o[w][q][d0 + j], acc[j]);
  }
  const int rr = row0 + q;
  if (p.nsplit == 1) {
    T* dst = reinterpret_cast<T*>(p.out) + (((long long)b * p.Tq + rr / G) * p.H + hkv * G + rr % G) * p.D;
    const float inv = (MODE != CONTIG || p.cap == 0) && L == 0.f ? 0.f : 1.f / L;     // no key at all: zeros
#pragma unroll
    for (int j = 0; j < VW; ++j)
      if (d0 + j < p.D) dst[d0 + j] = E::from_f32(acc[j] * inv);
  } else {
    const long long part = (((long long)b * p.Hkv + hkv) * p.nsplit + split) * p.rows + rr;
    float* w = p.ws + part * (DP + 2);
    if (d0 == 0) { w[DP] = M; w[DP + 1] = L; }
#pragma unroll
    for (int j = 0; j < VW; ++j) w[d0 + j] = acc[j];
  }
}

// One wave per query row: the parts of its splits (maximum, sum, unnormalised output) into one, eight at a time.  What a part's
// loads need is its number alone -- neither the sequence's length nor another part's maximum -- so that the launch costs one
// round trip to memory; parts that no workgroup wrote are dropped after the load.
template <typename T, int DP, bool PAGED>
__global__ __launch_bounds__(256) void decode_join_kernel(const DecodeArgs p) {
  constexpr int VW = DP < 64 ? 1 : DP / 64, N = 8;
  const int lane = threadIdx.x & 63, G = p.H / p.Hkv;
  const long long id = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (id >= (long long)p.B * p.Hkv * p.rows) return;
  const int rr = (int)(id % p.rows), hkv = (int)(id / p.rows % p.Hkv), b = (int)(id / ((long long)p.rows * p.Hkv));
  const float* w = p.ws + ((((long long)b * p.Hkv + hkv) * p.nsplit) * p.rows + rr) * (DP + 2);
  const long long step = (long long)p.rows * (DP + 2);
  const int d = min(lane * VW, DP - VW);
  int len = p.lens ? p.lens[b] : p.cap;
  float M = -INFINITY, L = 0.f, acc[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) acc[j] = 0.f;
  for (int s0 = 0; s0 < p.nsplit; s0 += N) {
    float m[N], l[N], o[N][VW];
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const float* part = w + min(s0 + s, p.nsplit - 1) * step;
      m[s] = part[DP];
      l[s] = part[DP + 1];
#pragma unroll
      for (int j = 0; j < VW; ++j) o[s][j] = part[d + j];
    }
    if (s0 == 0) {
      len = max(0, min(len, p.cap));
      if (!PAGED && len == 0) len = p.cap;
    }
    const int ns = max(1, (len + p.chunk - 1) / p.chunk);
    float mx = M;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      if (s0 + s >= ns) { m[s] = -INFINITY; l[s] = 0.f; }
      mx = attn_max(mx, m[s]);
    }
    const float base = mx == -INFINITY ? 0.f : mx, old = __builtin_amdgcn_exp2f(M - base);
    M = mx;
    L *= old;
#pragma unroll
    for (int j = 0; j < VW; ++j) acc[j] *= old;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const float f = __builtin_amdgcn_exp2f(m[s] - base);
      L = fmaf(f, l[s], L);
#pragma unroll
      for (int j = 0; j < VW; ++j) acc[j] = s0 + s < ns ? fmaf(f, o[s][j], acc[j]) : acc[j];
    }
    if (s0 + N >= ns) break;
  }
  const float inv = PAGED && L == 0.f ? 0.f : 1.f / L;
  T* out = reinterpret_cast<T*>(p.out) + (((long long)b * p.Tq + rr / G) * p.H + hkv * G + rr % G) * p.D;
#pragma unroll
  for (int j = 0; j < VW; ++j)
    if (lane * VW + j < p.D) out[lane * VW + j] = AttnElem<T>::from_f32(acc[j] * inv);
}

template <typename T, int DP>
int launch_decode(const DecodeArgs& p, hipStream_t st) {
  const dim3 grid((unsigned)p.nsplit, (unsigned)(p.Hkv * p.ngrp), (unsigned)p.B);
  if (!p.table) hipLaunchKernelGGL((decode_attn_kernel<T, DP, CONTIG>), grid, dim3(256), 0, st, p);
  else if (p.page % 16 == 0) hipLaunchKernelGGL((decode_attn_kernel<T, DP, BLOCK16>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((decode_attn_kernel<T, DP, ROWS>), grid, dim3(256), 0, st, p);
  NSP_LAUNCH_CHECK();
  if (p.nsplit > 1) {
    const dim3 jg((unsigned)(((long long)p.B * p.Hkv * p.rows + 3) / 4));
    if (p.table) hipLaunchKernelGGL((decode_join_kernel<T, DP, true>), jg, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((decode_join_kernel<T, DP, false>), jg, dim3(256), 0, st, p);
    NSP_LAUNCH_CHECK();
  }
  return NSP_OK;
}

template <typename T>
int launch_decode_d(const DecodeArgs& p, hipStream_t st) {
  if (p.D <= 32) return launch_decode<T, 32>(p, st);
  if (p.D <= 64) return launch_decode<T, 64>(p, st);
  return launch_decode<T, 128>(p, st);
}

// one 16-byte piece of a destination row per thread; grid.y = sequence
template <typename S, typename T>
__global__ __launch_bounds__(256) void paged_append_kernel(const S* __restrict__ k, const S* __restrict__ v, T* k_pages,
                                                           T* v_pages, const int* __restrict__ table,
                                                           const int* __restrict__ starts, const int* __restrict__ counts,
                                                           const nsp_paged_append_params a) {
  constexpr int CE = AttnElem<T>::CE;
  const int b = blockIdx.y, pieces = (int)a.D / CE;
  const int at0 = starts[b];
  const int n = counts ? min((int)a.n, counts[b]) : (int)a.n;
  const long long total = (long long)n * a.Hkv * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const int c = (int)(i % pieces), h = (int)(i / pieces % a.Hkv), t = (int)(i / ((long long)pieces * a.Hkv));
    const long long pos = (long long)at0 + t;
    if (at0 < 0 || pos >= (long long)a.width * a.page) continue;
    const int id = table[(long long)b * a.width + pos / a.page];
    if (id < 0 || id >= a.n_pages) continue;
    const long long slot = pos % a.page;
    const S* ks = k + (long long)b * a.k_sb + (long long)t * a.k_st + (long long)h * a.k_sh + c * CE;
    const S* vs = v + (long long)b * a.v_sb + (long long)t * a.v_st + (long long)h * a.v_sh + c * CE;
    T* kd = k_pages + id * a.kp_sp + slot * a.kp_ss + h * a.kp_sh + c * CE;
    T* vd = v_pages + id * a.vp_sp + slot * a.vp_ss + h * a.vp_sh + c * CE;
    typename AttnElem<T>::chunk x, y;
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      x[e] = (T)(float)ks[e];
      y[e] = (T)(float)vs[e];
    }
    *reinterpret_cast<typename AttnElem<T>::chunk*>(kd) = x;
    *reinterpret_cast<typename AttnElem<T>::chunk*>(vd) = y;
  }
}

// keys per workgroup and the number of workgroups a row of keys is split over
void decode_plan(long long groups, long long cap, int DP, int* nsplit, int* chunk) {
  // The chip holds 512 workgroups (d > 64) or 1024 at a time; four times as many even out sequences of unequal length, which
  // reach only part of the capacity that the call knows.  16 x 8 key heads, d 128, 9000..32000 of 32064 keys: 8 / 16 / 32 stretches
  // 282 / 274 / 294 us; 64 x 8, d 64, 700..1500 of 1500: 2 / 4 / 6 stretches 31.4 / 31.2 / 26.9 us.  No stretch is below 256 keys: a
  // workgroup's four waves then work through two tiles each; and up to 512 keys stay one: the second launch (3 us, and 4 us of the
  // host's time) costs more than it brings.
  long long want = ((DP == 128 ? 2048 : 4096) + groups - 1) / groups;
  const long long most = (cap + 255) / 256;
  if (want > most) want = most;
  if (want < 1 || cap <= 512) want = 1;
  long long c = (cap + want - 1) / want;
  c = (c + 127) / 128 * 128;
  if (c < 128) c = 128;
  *chunk = (int)c;
  *nsplit = (int)((cap + c - 1) / c);
  if (*nsplit < 1) *nsplit = 1;
}
int padded_head(long long D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

}  // namespace

extern "C" long long nsp_decode_attn_workspace_bytes(int B, int H, int Hkv, int Tq, int D, int cap) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || Tq <= 0 || D <= 0 || D > 128 || cap < 0) return 0;
  const long long rows = (long long)(H / Hkv) * Tq;
  int nsplit, chunk;
  const int DP = padded_head(D);
  decode_plan((long long)B * Hkv * ((rows + 15) / 16), cap, DP, &nsplit, &chunk);
  return nsplit == 1 ? 0 : (long long)B * Hkv * nsplit * rows * (DP + 2) * 4;
}

extern "C" int nsp_decode_attn(const nsp_decode_attn_params* a, void* stream) {
  if (!a || !a->q || !a->out) return NSP_EINVAL;
  if (a->B < 0 || a->Tq < 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->D <= 0) return NSP_EINVAL;
  if (a->D % 8 || a->D > 128 || (a->dtype != NSP_DT_F32 && a->dtype != NSP_DT_BF16)) return NSP_EUNSUPPORTED;
  if (a->B == 0 || a->Tq == 0) return NSP_OK;
  if (a->width < 0 || (a->table && (a->width == 0 || a->page <= 0 || a->n_pages < 0 || !a->lens)) || (!a->table && a->k_new)) return NSP_EINVAL;
  if ((a->k_new != nullptr) != (a->v_new != nullptr)) return NSP_EINVAL;
  const long long cap = a->table ? a->width * a->page : a->width;
  if (cap > 0 && (!a->k || !a->v)) return NSP_EINVAL;
  const long long rows = a->H / a->Hkv * a->Tq, ngrp = (rows + 15) / 16;
  // 32-bit key positions; grid dimensions
  if (cap > 0x7f000000LL || a->B > 65535 || a->Hkv * ngrp > 65535 || rows > 0x7fffffffLL) return NSP_EUNSUPPORTED;
  DecodeArgs p;
  p.q = a->q; p.out = a->out; p.k = a->k; p.v = a->v; p.table = a->table; p.lens = a->lens;
  p.k_new = a->k_new; p.v_new = a->v_new; p.ws = a->ws;
  p.B = (int)a->B; p.H = (int)a->H; p.Hkv = (int)a->Hkv; p.D = (int)a->D; p.Tq = (int)a->Tq;
  p.page = (int)a->page; p.n_pages = (unsigned)std::min(a->n_pages, 1LL << 31); p.width = (int)a->width;
  p.cap = (int)cap; p.rows = (int)rows; p.ngrp = (int)ngrp;
  p.page_magic = a->table ? (a->page == 1 ? 0xFFFFFFFFu : (unsigned)(0x100000000ULL / (unsigned long long)a->page)) : 0u;
  p.q_sb = a->q_sb; p.q_st = a->q_st; p.q_sh = a->q_sh;
  p.k_sp = a->k_sp; p.k_ss = a->k_ss; p.k_sh = a->k_sh;
  p.v_sp = a->v_sp; p.v_ss = a->v_ss; p.v_sh = a->v_sh;
  p.kn_sb = a->kn_sb; p.kn_sh = a->kn_sh; p.vn_sb = a->vn_sb; p.vn_sh = a->vn_sh;
  p.sl2 = (float)(a->scale * 1.4426950408889634);
  decode_plan(a->B * a->Hkv * ngrp, cap, padded_head(a->D), &p.nsplit, &p.chunk);
  if (p.nsplit > 1 && !p.ws) return NSP_EINVAL;
  return a->dtype == NSP_DT_BF16 ? launch_decode_d<__bf16>(p, (hipStream_t)stream) : launch_decode_d<float>(p, (hipStream_t)stream);
}

extern "C" int nsp_paged_append(const nsp_paged_append_params* a, void* stream) {
  if (!a || !a->k || !a->v || !a->k_pages || !a->v_pages || !a->table || !a->starts) return NSP_EINVAL;
  if (a->B < 0 || a->n < 0 || a->Hkv <= 0 || a->D <= 0 || a->page <= 0 || a->width < 0 || a->n_pages < 0) return NSP_EINVAL;
  if (a->D % 8 || a->D > 128 || a->B > 65535 || a->n > 0x7fffffffLL || a->width * a->page > 0x7f000000LL) return NSP_EUNSUPPORTED;
  if (a->B == 0 || a->n == 0 || a->width == 0) return NSP_OK;
  const long long pieces = a->D / (a->dtype == NSP_DT_BF16 ? 8 : 4);
  long long gx = (a->n * a->Hkv * pieces + 255) / 256;
  if (gx > 4096) gx = 4096;
  const dim3 grid((unsigned)gx, (unsigned)a->B);
  const hipStream_t st = (hipStream_t)stream;
#define NSP_APPEND(S, T)                                                                                             \
  hipLaunchKernelGGL((paged_append_kernel<S, T>), grid, dim3(256), 0, st, (const S*)a->k, (const S*)a->v, (T*)a->k_pages, \
                     (T*)a->v_pages, a->table, a->starts, a->counts, *a)
  if (a->src_dtype == NSP_DT_F32 && a->dtype == NSP_DT_F32) NSP_APPEND(float, float);
  else if (a->src_dtype == NSP_DT_F32 && a->dtype == NSP_DT_BF16) NSP_APPEND(float, __bf16);
  else if (a->src_dtype == NSP_DT_BF16 && a->dtype == NSP_DT_BF16) NSP_APPEND(__bf16, __bf16);
  else return NSP_EUNSUPPORTED;
#undef NSP_APPEND
  NSP_LAUNCH_CHECK();
  return NSP_OK;
}
