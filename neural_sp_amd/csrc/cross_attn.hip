// cross_attn.hip -- attention of target tokens over encoder states of another length, forward and backward.
//
//   S = scale Q K^T,  P = softmax over the keys j < klens[b],  O = dropout(P) V
//   dV = dropout(P)^T dO,  dP = dropout'(dO V^T),  D_i = sum_d dO_id O_id,  dS = P (dP - D),  dQ = scale dS K,  dK = scale dS^T Q
//
// No score leaves the compute unit.  All three kernels are one loop: a wave owns 16 rows (forward: 16 or 32) whose operands stay in
// registers, a workgroup of four waves streams tiles of the other side's rows through LDS (LDS-DMA, two or three pairs, one
// barrier per tile), and the score tile is computed with the OWNED row on the lane's column: row statistics are per lane, and
// the probabilities already are the operand of the second product -- their contraction runs over the streamed rows, four of
// which a lane holds per 16.
//   forward   owns queries, streams K and V;   O^T += V^T P^T
//   dQ        owns queries, streams K and V;   dQ^T += K^T dS^T; also D, which it leaves for
//   dK / dV   owns keys, streams Q and dO (of every query head of the key head: shared heads are summed in registers, in a
//             fixed order);                    dV^T += dO^T P, dK^T += Q^T dS
// The second operand of those products has the STREAMED row as contraction, i.e. wants a tile read across its rows: bf16 takes
// it with the transposing LDS read (ds_read_b64_tr_b16), fp32 holds one contraction element per lane and instruction and
// just picks the row.
// The softmax is kept as the forward pass's reference (log2 domain; the row's maximum or up to 8 below it, see there) and the
// reciprocal of the sum that goes with it, both fp32; backward recomputes P from them.
// bf16 roundings inside: P resp. dS, once each, as operands of the second products; with the outputs' own rounding the results are
// 1.2 (out) to 1.5 times (dQ) as far from exact as a rounding of the exact result.  (Two bf16 parts for dS bring dQ to 1.2 and cost
// 36 us of the 410 us of the largest measured call.)  Sums, statistics and D are fp32.
// A row without a visible key is uniform over all Tk keys, as with the finite mask value of attn_softmax_fwd, and passes no
// gradient through its scores.  Keys behind klens are never read.  What is not there (dimensions between the head size and the
// kernel's width, rows behind the last of a tile) enters as zeros on both sides, so infinities stay what the formulas make of them:
// a key with a score of -inf has no probability, an infinite value makes infinite sums.
#include "attn_frag.h"
#include <type_traits>

namespace {

struct XArgs {
  const void *q, *k, *v, *dout;
  void *out, *dq, *dk, *dv;
  float* stats;        // [2][B,H,Tq]: the exponents' reference, 1 / sum
  float* rows;         // [3][B,H,Tq rounded up to 64]: what dK / dV need of every query, from the dQ kernel
  const int* klens;
  int B, H, Hkv, D, Tq, Tk;
  long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, g_sb, g_st, g_sh;
  unsigned long long seed, offset;
  float scale, sl2, drop;
};

typedef __attribute__((address_space(3))) bf16x4 x_lds_bf16x4;
typedef __attribute__((address_space(3))) void x_lds_void;
typedef const __attribute__((address_space(1))) void x_glb_void;

// ---- a tile: KT rows of DP elements, 16-byte chunks XOR-swizzled by the row (unpadded: the DMA writes lane-linear)
template <typename T, int DP>
struct XTile {
  typedef AttnElem<T> E;
  static constexpr int KT = sizeof(T) == 2 ? 64 : 32;
  static constexpr int RB = DP * (int)sizeof(T);     // bytes of a row
  static constexpr int CPR = RB / 16;                // chunks of a row
  static constexpr int NS = CPR / 4;                 // steps of a product over the head size
  static constexpr int NB = DP / 16;                 // 16-row blocks of a transposed accumulator
  static constexpr int BYTES = KT * RB;
  static constexpr int U = KT / 32;                  // 32-row steps of a tile
  static constexpr int HALF = 32 * RB;
  // pairs of tiles in LDS: with three, two are on their way while one is worked on (48 KB and three workgroups per compute unit);
  // the 128-wide pairs are too large for that
  static constexpr int STAGES = DP <= 64 ? 3 : 2;
  __device__ static __forceinline__ int swz(int row) { return RB >= 128 ? (row & 7) : ((row >> 1) & 3); }
  // operand of a product over the head size: chunk 4 s + g of row rbase + r
  __device__ static __forceinline__ typename E::chunk rows(const unsigned char* tile, int rbase, int s, int r, int g) {
    const int row = rbase + r;
    return *reinterpret_cast<const typename E::chunk*>(tile + row * RB + (((4 * s + g) ^ swz(row)) << 4));
  }
};

// where a workgroup's tiles come from: a uniform address per tile and 32-bit offsets per lane that stay (strides below 2^24
// elements), so that the requests of a tile cost no vector arithmetic.  What a tile has and the source has not (chunks behind a
// head size below DP, rows behind the last) is read from 16 bytes of zeros: the other operand is 0 there as well, and 0 times a
// copy of another element would be NaN where that is infinite.  Every lane takes part in every request, so their number per wave
// stays the same.
__device__ const nsp_u32x4 x_zeros = {0u, 0u, 0u, 0u};
template <typename T, int DP>
struct XSource {
  typedef XTile<T, DP> X;
  static constexpr int P = X::BYTES / 4096;          // instructions (1 KB each) of a wave
  const unsigned char* base;
  unsigned ldb, off[P];
  int wave, lane, chunks;      // (chunks of a source row)
  __device__ __forceinline__ int row_of(int i, int l) const { return (wave * P + i) * (64 / X::CPR) + l / X::CPR; }
  __device__ __forceinline__ int chunk_of(int i, int l) const { return l % X::CPR ^ X::swz(row_of(i, l)); }
  __device__ __forceinline__ void init(const T* src, long long ld, int chunks_, int wave_, int lane_) {
    base = reinterpret_cast<const unsigned char*>(src);
    ldb = (unsigned)ld * (unsigned)sizeof(T);
    wave = wave_;
    lane = lane_;
    chunks = chunks_;
#pragma unroll
    for (int i = 0; i < P; ++i) off[i] = (unsigned)row_of(i, lane) * ldb + (unsigned)chunk_of(i, lane) * 16u;
  }
  // rows row0 .. row0 + KT - 1 into LDS; rows from `limit` (> row0) on are zeros, or (AGAIN) the last one again
  template <bool AGAIN>
  __device__ __forceinline__ void request(unsigned char* tile, long long skip, int row0, int limit) const {
    const unsigned char* at = base + skip + (long long)row0 * ldb;
    if (row0 + X::KT <= limit && chunks == X::CPR) {
#pragma unroll
      for (int i = 0; i < P; ++i)
        __builtin_amdgcn_global_load_lds((x_glb_void*)(at + off[i]), (x_lds_void*)(tile + (wave * P + i) * 1024), 16, 0, 0);
    } else {
      int l = lane;
#ifndef NSP_HOST_EMULATION
      asm volatile("" : "+v"(l));      // (computed here: held over the loop it would cost a dozen registers)
#endif
      const int last = limit - 1 - row0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int chunk = chunk_of(i, l);
        const bool behind = row_of(i, l) > last;
        const unsigned char* from = at + (AGAIN && behind ? (unsigned)last * ldb + (unsigned)chunk * 16u : off[i]);
        if (chunk >= chunks || (!AGAIN && behind)) from = reinterpret_cast<const unsigned char*>(&x_zeros);
        __builtin_amdgcn_global_load_lds((x_glb_void*)from, (x_lds_void*)(tile + (wave * P + i) * 1024), 16, 0, 0);
      }
    }
  }
};

// ---- 32 rows of a tile as the operand of a product that runs over these rows:
//   acc[f][blk] (rows: 16 dimensions, column: owned row) += sum over the rows  row^T w,  w[f][kf][e] = weight of row 16 kf + 4 g + e
template <typename T, int DP>
struct XAcross;

// fp32: a lane holds one contraction element per instruction and picks its row: dimension blk of row m is m * DP / 16 + blk
template <int DP>
struct XAcross<float, DP> {
  typedef XTile<float, DP> X;
  static constexpr int VW = DP / 16;
  template <int OFF>
  __device__ __forceinline__ void read(const unsigned char*, const unsigned*) {}
  template <int OA, int OB>
  __device__ static __forceinline__ void read2(XAcross&, XAcross&, const unsigned char*, const unsigned*) {}
  template <int OFF, bool SUM, int N>
  __device__ __forceinline__ void product(f32x4 (&acc)[N][VW], f32x4 (&)[N], const f32x4 (&w)[N][2], const unsigned char* lds, int r,
                                          int g) const {
#pragma unroll
    for (int kf = 0; kf < 2; ++kf)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * kf + 4 * g + e;
        const float* base = reinterpret_cast<const float*>(lds + OFF + row * X::RB);
        float x[VW];
#pragma unroll
        for (int i = 0; i < VW; i += (VW < 4 ? VW : 4)) {
          const int el = r * VW + i, c = el >> 2;
          const float* p = base + ((c ^ X::swz(row)) << 2) + (el & 3);
          if constexpr (VW == 2) {
            const float2 a = *reinterpret_cast<const float2*>(p);
            x[0] = a.x; x[1] = a.y;
          } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i + j] = a[j];
          }
        }
#pragma unroll
        for (int f = 0; f < N; ++f)
#pragma unroll
          for (int j = 0; j < VW; ++j) acc[f][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], w[f][kf][e], acc[f][j], 0, 0, 0);
      }
  }
};

// bf16: transposing LDS reads, dimension blk of row m is 16 blk + m.  The reads and their wait are ONE statement, so that no other
// instruction can touch a destination in between.  (The builtin is modelled as reading memory that an LDS-DMA in flight may
// write: hipcc would wait for the next tile's DMA in front of it.)  The statement's wait hides behind the matrix instructions
// issued before it: the callers put it between the score products and what needs their results.  A lane has one address per
// 16 dimensions (of the first 64: the swizzle leaves 128-byte steps alone); rows, tiles and buffers are offsets in the instruction.
template <int DP>
__device__ __forceinline__ void x_tr_addr(unsigned (&ta)[4], const unsigned char* lds, int r, int g) {
  typedef XTile<__bf16, DP> X;
  const int row = 4 * g + (r >> 2), b = r & 3;
#ifdef NSP_HOST_EMULATION
  const unsigned at = 0;
#else
  typedef __attribute__((address_space(3))) unsigned char lds_uchar;
  const unsigned at = (unsigned)(uintptr_t)((lds_uchar*)const_cast<unsigned char*>(lds));
#endif
#pragma unroll
  for (int i = 0; i < (DP == 32 ? 2 : 4); ++i)
    ta[i] = at + (unsigned)(row * X::RB + (((2 * i + (b >> 1)) ^ X::swz(row)) << 4) + (b & 1) * 8);
}
// 4 + 4 fragments of 32 rows x 16 dimensions at byte offsets OA and OB
template <int OA, int OB, int RB>
__device__ __forceinline__ void x_tr_read16(bf16x8* a, bf16x8* b, const unsigned char* lds, const unsigned* ta) {
  bf16x4 al[4], ah[4], bl[4], bh[4];
#ifdef NSP_HOST_EMULATION
  for (int i = 0; i < 4; ++i) {
    al[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OA));
    ah[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OA + 16 * RB));
    bl[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OB));
    bh[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OB + 16 * RB));
  }
#else
  (void)lds;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16 offset:%20\n\tds_read_b64_tr_b16 %1, %16 offset:%21\n\t"
      "ds_read_b64_tr_b16 %2, %17 offset:%20\n\tds_read_b64_tr_b16 %3, %17 offset:%21\n\t"
      "ds_read_b64_tr_b16 %4, %18 offset:%20\n\tds_read_b64_tr_b16 %5, %18 offset:%21\n\t"
      "ds_read_b64_tr_b16 %6, %19 offset:%20\n\tds_read_b64_tr_b16 %7, %19 offset:%21\n\t"
      "ds_read_b64_tr_b16 %8, %16 offset:%22\n\tds_read_b64_tr_b16 %9, %16 offset:%23\n\t"
      "ds_read_b64_tr_b16 %10, %17 offset:%22\n\tds_read_b64_tr_b16 %11, %17 offset:%23\n\t"
      "ds_read_b64_tr_b16 %12, %18 offset:%22\n\tds_read_b64_tr_b16 %13, %18 offset:%23\n\t"
      "ds_read_b64_tr_b16 %14, %19 offset:%22\n\tds_read_b64_tr_b16 %15, %19 offset:%23\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(al[0]), "=&v"(ah[0]), "=&v"(al[1]), "=&v"(ah[1]), "=&v"(al[2]), "=&v"(ah[2]), "=&v"(al[3]), "=&v"(ah[3]),
        "=&v"(bl[0]), "=&v"(bh[0]), "=&v"(bl[1]), "=&v"(bh[1]), "=&v"(bl[2]), "=&v"(bh[2]), "=&v"(bl[3]), "=&v"(bh[3])
      : "v"(ta[0]), "v"(ta[1]), "v"(ta[2]), "v"(ta[3]), "i"(OA), "i"(OA + 16 * RB), "i"(OB), "i"(OB + 16 * RB)
      : "memory");
#endif
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = __builtin_shufflevector(al[i], ah[i], 0, 1, 2, 3, 4, 5, 6, 7);
    b[i] = __builtin_shufflevector(bl[i], bh[i], 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
template <int OFF, int RB>
__device__ __forceinline__ void x_tr_read8(bf16x8* out, const unsigned char* lds, const unsigned* ta) {
  bf16x4 lo[4], hi[4];
#ifdef NSP_HOST_EMULATION
  for (int i = 0; i < 4; ++i) {
    lo[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OFF));
    hi[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OFF + 16 * RB));
  }
#else
  (void)lds;
  asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
               "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
               "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
               "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
               : "v"(ta[0]), "v"(ta[1]), "v"(ta[2]), "v"(ta[3]), "i"(OFF), "i"(OFF + 16 * RB)
               : "memory");
#endif
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int OFF, int RB>
__device__ __forceinline__ void x_tr_read4(bf16x8* out, const unsigned char* lds, const unsigned* ta) {
  bf16x4 lo[2], hi[2];
#ifdef NSP_HOST_EMULATION
  for (int i = 0; i < 2; ++i) {
    lo[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OFF));
    hi[i] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((x_lds_bf16x4*)(lds + ta[i] + OFF + 16 * RB));
  }
#else
  (void)lds;
  asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
               "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
               : "v"(ta[0]), "v"(ta[1]), "i"(OFF), "i"(OFF + 16 * RB)
               : "memory");
#endif
#pragma unroll
  for (int i = 0; i < 2; ++i) out[i] = __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int DP>
struct XAcross<__bf16, DP> {
  typedef XTile<__bf16, DP> X;
  bf16x8 t[X::NB];
  template <int OFF>
  __device__ __forceinline__ void read(const unsigned char* lds, const unsigned* ta) {
    if constexpr (DP == 32) x_tr_read4<OFF, X::RB>(t, lds, ta);
    else if constexpr (DP == 64) x_tr_read8<OFF, X::RB>(t, lds, ta);
    else x_tr_read16<OFF, OFF + 128, X::RB>(t, t + 4, lds, ta);
  }
  template <int OA, int OB>
  __device__ static __forceinline__ void read2(XAcross& a, XAcross& b, const unsigned char* lds, const unsigned* ta) {
    if constexpr (DP == 64) {
      x_tr_read16<OA, OB, X::RB>(a.t, b.t, lds, ta);
    } else {
      a.template read<OA>(lds, ta);
      b.template read<OB>(lds, ta);
    }
  }
  // SUM: sum[f] (every element) += the column's weights as they enter, by a product with ones -- the matrix cores have more room
  // for it than the vector units
  template <int OFF, bool SUM, int N>
  __device__ __forceinline__ void product(f32x4 (&acc)[N][X::NB], f32x4 (&sum)[N], const f32x4 (&w)[N][2], const unsigned char*, int,
                                          int) const {
    bf16x8 p[N];
#pragma unroll
    for (int f = 0; f < N; ++f)
#pragma unroll
      for (int i = 0; i < 8; ++i) p[f][i] = (__bf16)w[f][i >> 2][i & 3];
    if constexpr (SUM) {
      bf16x8 one;
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = (__bf16)1.f;
#pragma unroll
      for (int f = 0; f < N; ++f) sum[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(one, p[f], sum[f], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < X::NB; ++i)
#pragma unroll
      for (int f = 0; f < N; ++f) acc[f][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(t[i], p[f], acc[f][i], 0, 0, 0);
  }
};

// row `dst` (D elements) <- a transposed accumulator's column, times f
template <int DP>
__device__ __forceinline__ void x_store(float* dst, const f32x4 (&acc)[DP / 16], float f, int D, int g) {
  constexpr int VW = DP / 16;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = (4 * g + e) * VW;
    if (d >= D) continue;
    if constexpr (VW == 2) {
      *reinterpret_cast<float2*>(dst + d) = make_float2(acc[0][e] * f, acc[1][e] * f);
    } else {
#pragma unroll
      for (int i = 0; i < VW; i += 4)
        *reinterpret_cast<f32x4*>(dst + d + i) = f32x4{acc[i][e] * f, acc[i + 1][e] * f, acc[i + 2][e] * f, acc[i + 3][e] * f};
    }
  }
}
template <int DP>
__device__ __forceinline__ void x_store(__bf16* dst, const f32x4 (&acc)[DP / 16], float f, int D, int g) {
#pragma unroll
  for (int blk = 0; blk < DP / 16; ++blk) {
    const int d = 16 * blk + 4 * g;
    if (d >= D) continue;
    bf16x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = (__bf16)(acc[blk][e] * f);
    }
    *reinterpret_cast<bf16x4*>(dst + d) = x;
  }
}

// which (sequence, key head, query head of the group, row tile) a workgroup takes: workgroups go round the eight XCDs in
// turn, and all the ones that stream the same rows are put on one of them, one after the other
__device__ __forceinline__ bool x_place(int groups, int per, int& grp, int& item) {
  const int id = (int)blockIdx.x, i = id >> 3;
  grp = (i / per) * 8 + (id & 7);
  item = i % per;
  return grp < groups;
}

template <typename T, int N, int NS>
__device__ __forceinline__ void x_load_rows(typename AttnElem<T>::chunk (&f)[N][NS], const T* base, long long ld, int row0,
                                            int limit, int D, int r, int g) {
  typedef AttnElem<T> E;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const T* p = base + (long long)min(row0 + 16 * i + r, limit - 1) * ld;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int c = (4 * s + g) * E::CE;
      f[i][s] = c < D ? *reinterpret_cast<const typename E::chunk*>(p + c) : E::zero();
    }
  }
}

// scores of 32 streamed rows: s[f][kf] rows = streamed rows 16 kf + 4 g + e, column = owned row; init(f, kf) is added (the matrix
// instruction's accumulator starts with it)
template <typename T, int DP, int N, int NS, class I>
__device__ __forceinline__ void x_product(f32x4 (&s)[N][2], const unsigned char* tile,
                                          const typename AttnElem<T>::chunk (&own)[N][NS], int r, int g, I init) {
  typedef XTile<T, DP> X;
#pragma unroll
  for (int kf = 0; kf < 2; ++kf) {
#pragma unroll
    for (int f = 0; f < N; ++f) s[f][kf] = init(f, kf);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const auto a = X::rows(tile, 16 * kf, i, r, g);
#pragma unroll
      for (int f = 0; f < N; ++f) s[f][kf] = AttnElem<T>::mma(a, own[f][i], s[f][kf]);
    }
  }
}
// Behind the last read of a tile: the next one has landed (all but the newest `NEWER` requests of the wave are done; `last`: all)
// and every wave has read this one.  A bare barrier: the fence of __syncthreads would wait for the tiles still on their way.
template <int NEWER>
__device__ __forceinline__ void x_turn(bool last) {
  if (NEWER > 0 && !last) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NEWER) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct XZero {
  __device__ __forceinline__ f32x4 operator()(int, int) const { return f32x4{0.f, 0.f, 0.f, 0.f}; }
};

template <typename T, int DP, int NQ, bool DROP>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void cross_fwd_kernel(const XArgs p) {
  typedef XTile<T, DP> X;
  __shared__ __attribute__((aligned(16))) unsigned char lds[X::STAGES * 2 * X::BYTES];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int G = p.H / p.Hkv, nqt = (p.Tq + 64 * NQ - 1) / (64 * NQ);
  int grp, item;
  if (!x_place(p.B * p.Hkv, G * nqt, grp, item)) return;
  const int b = grp / p.Hkv, hkv = grp % p.Hkv, h = hkv * G + item / nqt;
  const int q0 = (item % nqt) * (64 * NQ) + wave * (16 * NQ);
  int klen = p.klens ? min(p.klens[b], p.Tk) : p.Tk;
  const bool uniform = klen <= 0;
  if (uniform) klen = p.Tk;
  const T* kb = reinterpret_cast<const T*>(p.k) + (long long)b * p.k_sb + (long long)hkv * p.k_sh;
  const T* vb = reinterpret_cast<const T*>(p.v) + (long long)b * p.v_sb + (long long)hkv * p.v_sh;
  const int chunks = p.D / X::E::CE;
  typename X::E::chunk Q[NQ][X::NS];
  x_load_rows<T, NQ>(Q, reinterpret_cast<const T*>(p.q) + (long long)b * p.q_sb + (long long)h * p.q_sh, p.q_st, q0, p.Tq,
                         p.D, r, g);
  constexpr bool SUM = sizeof(T) == 2 && !DROP;
  f32x4 o[NQ][X::NB], sum[NQ];
  float m[NQ], l[NQ];
#pragma unroll
  for (int f = 0; f < NQ; ++f) {
#pragma unroll
    for (int i = 0; i < X::NB; ++i) o[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    sum[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[f] = -3.4028235e38f;      // (finite: a tile whose scores are all -inf leaves the row as it is)
    l[f] = 0.f;
  }
  unsigned ta[4];
  if constexpr (sizeof(T) == 2) x_tr_addr<DP>(ta, lds, r, g);
  XSource<T, DP> ks, vs;
  ks.init(kb, p.k_st, chunks, wave, lane);
  vs.init(vb, p.v_st, chunks, wave, lane);
  const int nkt = (klen + X::KT - 1) / X::KT;
  constexpr int PAIR = 2 * X::BYTES, AHEAD = X::STAGES - 1, NEWER = (AHEAD - 1) * 2 * XSource<T, DP>::P;
  auto fetch = [&](int at, int kt) {
    ks.template request<false>(lds + at, 0, kt * X::KT, klen);
    vs.template request<false>(lds + at + X::BYTES, 0, kt * X::KT, klen);
  };
  fetch(0, 0);
  if (AHEAD > 1 && nkt > 1) fetch(PAIR, 1);
  x_turn<NEWER>(nkt <= AHEAD - 1);
  auto step = [&](int kt, auto BUF) {
    constexpr int AT = decltype(BUF)::value * PAIR, NEXT = (decltype(BUF)::value + AHEAD) % X::STAGES * PAIR;
    const unsigned char* Kc = lds + AT;
    // (that buffer was last read in step kt - 1, behind that step's barrier)
    if (kt + AHEAD < nkt) fetch(NEXT, kt + AHEAD);
    f32x4 s[X::U][NQ][2];
#pragma unroll
    for (int u = 0; u < X::U; ++u) x_product<T, DP, NQ>(s[u], Kc + u * X::HALF, Q, r, g, XZero());
    __builtin_amdgcn_sched_barrier(0);      // (the products are under way while the values are read)
    XAcross<T, DP> v[X::U];
    if constexpr (X::U == 2) XAcross<T, DP>::template read2<AT + X::BYTES, AT + X::BYTES + X::HALF>(v[0], v[X::U - 1], lds, ta);
    __builtin_amdgcn_sched_barrier(0);
    if (uniform || (kt + 1) * X::KT > klen) {
#pragma unroll
      for (int u = 0; u < X::U; ++u)
#pragma unroll
        for (int f = 0; f < NQ; ++f)
#pragma unroll
          for (int kf = 0; kf < 2; ++kf)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (uniform) s[u][f][kf][e] = 0.f;
              if (kt * X::KT + 32 * u + 16 * kf + 4 * g + e >= klen) s[u][f][kf][e] = -INFINITY;
            }
    }
    // The reference maximum moves only when a score exceeds it by 2^8: exponentials then stay below 2^8 (exact in range for both
    // types, and bf16 keeps its relative precision), and after the first tiles nothing is rescaled any more.
    float mx[NQ];
    bool move = false;
#pragma unroll
    for (int f = 0; f < NQ; ++f) {
      mx[f] = s[0][f][0][0];
#pragma unroll
      for (int u = 0; u < X::U; ++u)
#pragma unroll
        for (int kf = 0; kf < 2; ++kf)
          mx[f] = attn_max(attn_max(attn_max(mx[f], s[u][f][kf][0]), attn_max(s[u][f][kf][1], s[u][f][kf][2])), s[u][f][kf][3]);
      mx[f] = attn_max4(mx[f]) * p.sl2;    // (scale > 0: the maximum commutes with it)
      move = move || !(mx[f] <= m[f] + 8.f);
    }
    if (__any(move)) {
#pragma unroll
      for (int f = 0; f < NQ; ++f) {
        const float mn = attn_max(m[f], mx[f]);
        const float alpha = __builtin_amdgcn_exp2f(m[f] - mn);
        m[f] = mn;
        l[f] *= alpha;
        sum[f] *= alpha;
#pragma unroll
        for (int i = 0; i < X::NB; ++i) o[f][i] *= alpha;
      }
    }
#pragma unroll
    for (int f = 0; f < NQ; ++f) {
      const int qi = min(q0 + 16 * f + r, p.Tq - 1);
      const unsigned long long row =
          DROP ? p.offset + (unsigned long long)((((long long)b * p.H + h) * p.Tq + qi) * p.Tk) : 0ull;
#pragma unroll
      for (int u = 0; u < X::U; ++u)
#pragma unroll
        for (int kf = 0; kf < 2; ++kf) {
          float keep[4];
          if constexpr (DROP)
            nsp_keep_scale4(p.seed, row + (unsigned long long)(kt * X::KT + 32 * u + 16 * kf + 4 * g), p.drop, keep);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[u][f][kf][e], p.sl2, -m[f]));
            if constexpr (!SUM) l[f] += x;
            s[u][f][kf][e] = DROP ? x * keep[e] : x;
          }
        }
    }
    v[0].template product<AT + X::BYTES, SUM, NQ>(o, sum, s[0], lds, r, g);
    if constexpr (X::U == 2) v[1].template product<AT + X::BYTES + X::HALF, SUM, NQ>(o, sum, s[1], lds, r, g);
    x_turn<NEWER>(kt + AHEAD >= nkt);
  };
  for (int kt = 0; kt < nkt; kt += X::STAGES) {
    step(kt, std::integral_constant<int, 0>());
    if (kt + 1 < nkt) step(kt + 1, std::integral_constant<int, 1>());
    if constexpr (X::STAGES == 3)
      if (kt + 2 < nkt) step(kt + 2, std::integral_constant<int, 2>());
  }
#pragma unroll
  for (int f = 0; f < NQ; ++f) {
    const float inv = 1.f / (SUM ? sum[f][0] : attn_sum4(l[f]));
    const int qi = q0 + 16 * f + r;
    if (qi >= p.Tq) continue;
    const long long at = (((long long)b * p.Tq + qi) * p.H + h) * p.D;
    x_store<DP>(reinterpret_cast<T*>(p.out) + at, o[f], inv, p.D, g);
    if (p.stats && g == 0) {
      const long long sr = ((long long)b * p.H + h) * p.Tq + qi;
      p.stats[sr] = m[f];
      p.stats[(long long)p.B * p.H * p.Tq + sr] = inv;
    }
  }
}

template <typename T, int DP, bool DROP>
__global__ __launch_bounds__(256, 2) void cross_dq_kernel(const XArgs p) {
  typedef XTile<T, DP> X;
  constexpr int NQ = 1;      // owned 16-query fragments of a wave
  __shared__ __attribute__((aligned(16))) unsigned char lds[X::STAGES * 2 * X::BYTES];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int G = p.H / p.Hkv, nqt = (p.Tq + 64 * NQ - 1) / (64 * NQ);
  int grp, item;
  if (!x_place(p.B * p.Hkv, G * nqt, grp, item)) return;
  const int b = grp / p.Hkv, hkv = grp % p.Hkv, h = hkv * G + item / nqt;
  const int q0 = (item % nqt) * (64 * NQ) + wave * (16 * NQ);
  const int klen = p.klens ? min(p.klens[b], p.Tk) : p.Tk;
  const T* kb = reinterpret_cast<const T*>(p.k) + (long long)b * p.k_sb + (long long)hkv * p.k_sh;
  const T* vb = reinterpret_cast<const T*>(p.v) + (long long)b * p.v_sb + (long long)hkv * p.v_sh;
  const int chunks = p.D / X::E::CE;
  const long long srow = ((long long)b * p.H + h) * p.Tq;
  const int nkt = klen <= 0 ? 0 : (klen + X::KT - 1) / X::KT;     // no visible key: no gradient
  unsigned ta[4];
  // bf16: O was rounded, and so were the probabilities in it, so D is a little off.  The probabilities sum to 1, hence D is what is used
  // for it here plus the sum of dS, and what that changes is that sum times sum_j p_j k_j: both are kept and settled at the end.
  constexpr bool MEND = sizeof(T) == 2;
  float off[NQ];
  f32x4 pk[MEND ? NQ : 1][X::NB], none[NQ];
  if constexpr (sizeof(T) == 2) x_tr_addr<DP>(ta, lds, r, g);
  XSource<T, DP> ks, vs;
  ks.init(kb, p.k_st, chunks, wave, lane);
  vs.init(vb, p.v_st, chunks, wave, lane);
  constexpr int PAIR = 2 * X::BYTES, AHEAD = X::STAGES - 1, NEWER = (AHEAD - 1) * 2 * XSource<T, DP>::P;
  auto fetch = [&](int at, int kt) {
    ks.template request<false>(lds + at, 0, kt * X::KT, klen);
    vs.template request<false>(lds + at + X::BYTES, 0, kt * X::KT, klen);
  };
  if (nkt > 0) fetch(0, 0);
  typename X::E::chunk Q[NQ][X::NS], dO[NQ][X::NS];
  x_load_rows<T, NQ>(Q, reinterpret_cast<const T*>(p.q) + (long long)b * p.q_sb + (long long)h * p.q_sh, p.q_st, q0, p.Tq,
                         p.D, r, g);
  x_load_rows<T, NQ>(dO, reinterpret_cast<const T*>(p.dout) + (long long)b * p.g_sb + (long long)h * p.g_sh, p.g_st, q0,
                         p.Tq, p.D, r, g);
  float m[NQ], inv[NQ], ds[NQ];
  f32x4 acc[NQ][X::NB];
  {
    const long long orow = (long long)b * p.Tq * p.H * p.D + (long long)h * p.D;
#pragma unroll
    for (int f = 0; f < NQ; ++f) {
      typename X::E::chunk O[1][X::NS];
      float d = 0.f;
      x_load_rows<T, 1>(O, reinterpret_cast<const T*>(p.out) + orow, (long long)p.H * p.D, q0 + 16 * f, p.Tq, p.D, r, g);
#pragma unroll
      for (int s = 0; s < X::NS; ++s)
#pragma unroll
        for (int e = 0; e < X::E::CE; ++e) d = fmaf((float)dO[f][s][e], (float)O[0][s][e], d);
      ds[f] = attn_sum4(d);
      const int qi = min(q0 + 16 * f + r, p.Tq - 1);
      m[f] = p.stats[srow + qi];
      inv[f] = p.stats[(long long)p.B * p.H * p.Tq + srow + qi];
      if constexpr (sizeof(T) == 2) m[f] -= __log2f(inv[f]);      // (one rounding of the exponent more, far below bf16's)
      off[f] = 0.f;
      if constexpr (MEND) {
#pragma unroll
        for (int i = 0; i < X::NB; ++i) pk[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int i = 0; i < X::NB; ++i) acc[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  x_turn<0>(true);
  if (AHEAD > 1 && nkt > 1) fetch(PAIR, 1);
  auto step = [&](int kt, auto BUF) {
    constexpr int AT = decltype(BUF)::value * PAIR, NEXT = (decltype(BUF)::value + AHEAD) % X::STAGES * PAIR;
    if (kt + AHEAD < nkt) fetch(NEXT, kt + AHEAD);
    auto rows32 = [&](auto UC) {
      constexpr int u = decltype(UC)::value, R = AT + u * X::HALF;
      f32x4 s[NQ][2], dp[NQ][2];
      x_product<T, DP, NQ>(s, lds + R, Q, r, g, XZero());
      // dP - D in one go (with dropout D comes after the mask)
      x_product<T, DP, NQ>(dp, lds + R + X::BYTES, dO, r, g, [&](int f, int) -> f32x4 {
        return DROP ? f32x4{0.f, 0.f, 0.f, 0.f} : f32x4{-ds[f], -ds[f], -ds[f], -ds[f]};
      });
      __builtin_amdgcn_sched_barrier(0);
      XAcross<T, DP> k;
      k.template read<R>(lds, ta);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < NQ; ++f) {
        const int qi = min(q0 + 16 * f + r, p.Tq - 1);
        const unsigned long long row = DROP ? p.offset + (unsigned long long)((srow + qi) * p.Tk) : 0ull;
#pragma unroll
        for (int kf = 0; kf < 2; ++kf) {
          float keep[4];
          if constexpr (DROP)
            nsp_keep_scale4(p.seed, row + (unsigned long long)(kt * X::KT + 32 * u + 16 * kf + 4 * g), p.drop, keep);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = __builtin_amdgcn_exp2f(fmaf(s[f][kf][e], p.sl2, -m[f]));
            if constexpr (!MEND) x *= inv[f];
            s[f][kf][e] = x;
            if constexpr (DROP) dp[f][kf][e] = fmaf(dp[f][kf][e], keep[e], -ds[f]);
          }
        }
      }
      if (kt * X::KT + 32 * (u + 1) > klen) {
#pragma unroll
        for (int f = 0; f < NQ; ++f)
#pragma unroll
          for (int kf = 0; kf < 2; ++kf)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (kt * X::KT + 32 * u + 16 * kf + 4 * g + e >= klen) s[f][kf][e] = 0.f;
      }
#pragma unroll
      for (int f = 0; f < NQ; ++f)
#pragma unroll
        for (int kf = 0; kf < 2; ++kf) {
          dp[f][kf] *= s[f][kf];
          if constexpr (MEND) off[f] += (dp[f][kf][0] + dp[f][kf][1]) + (dp[f][kf][2] + dp[f][kf][3]);
        }
      k.template product<R, false, NQ>(acc, none, dp, lds, r, g);
      if constexpr (MEND) k.template product<R, false, NQ>(pk, none, s, lds, r, g);
    };
    rows32(std::integral_constant<int, 0>());
    if constexpr (X::U == 2) rows32(std::integral_constant<int, 1>());
    x_turn<NEWER>(kt + AHEAD >= nkt);
  };
  for (int kt = 0; kt < nkt; kt += X::STAGES) {
    step(kt, std::integral_constant<int, 0>());
    if (kt + 1 < nkt) step(kt + 1, std::integral_constant<int, 1>());
    if constexpr (X::STAGES == 3)
      if (kt + 2 < nkt) step(kt + 2, std::integral_constant<int, 2>());
  }
  // D and the statistics for the dK / dV kernel, which reads 64 at a time: rows behind the last query have probability 0
  const int pitch = (p.Tq + 63) / 64 * 64;
#pragma unroll
  for (int f = 0; f < NQ; ++f) {
    if constexpr (MEND) {
      off[f] = attn_sum4(off[f]);
#pragma unroll
      for (int i = 0; i < X::NB; ++i) acc[f][i] -= off[f] * pk[f][i];
    }
    const int q = q0 + 16 * f + r;
    if (g == 0 && q < pitch) {
      const long long at = ((long long)b * p.H + h) * pitch + q, n = (long long)p.B * p.H * pitch;
      p.rows[at] = q < p.Tq ? m[f] : INFINITY;
      p.rows[n + at] = q < p.Tq ? inv[f] : 0.f;
      p.rows[2 * n + at] = q < p.Tq ? ds[f] + off[f] : 0.f;
    }
    if (q < p.Tq)
      x_store<DP>(reinterpret_cast<T*>(p.dq) + (((long long)b * p.Tq + q) * p.H + h) * p.D, acc[f], p.scale, p.D, g);
  }
}

template <typename T, int DP, bool DROP>
__global__ __launch_bounds__(256, 2) void cross_dkv_kernel(const XArgs p) {
  typedef XTile<T, DP> X;
  constexpr int NK = 1;      // owned 16-key fragments of a wave
  // pairs of tiles, then for each the rows' maxima, reciprocal sums and D (64 each)
  // (two pairs: a fourth workgroup per compute unit is worth more than a third tile, 199 against 210 us)
  constexpr int STAGES = 2, PAIR = 2 * X::BYTES, ROWS = STAGES * PAIR;
  __shared__ __attribute__((aligned(16))) unsigned char lds[ROWS + STAGES * 1024];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int G = p.H / p.Hkv, nkt = (p.Tk + 64 * NK - 1) / (64 * NK);
  int grp, item;
  if (!x_place(p.B * p.Hkv, nkt, grp, item)) return;
  const int b = grp / p.Hkv, hkv = grp % p.Hkv;
  int klen = p.klens ? min(p.klens[b], p.Tk) : p.Tk;
  const bool uniform = klen <= 0;
  if (uniform) klen = p.Tk;
  const int k0 = (item * 4 + wave) * (16 * NK);
  f32x4 dk[NK][X::NB], dv[NK][X::NB];
#pragma unroll
  for (int f = 0; f < NK; ++f)
#pragma unroll
    for (int i = 0; i < X::NB; ++i) dk[f][i] = dv[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (item * (64 * NK) < klen) {      // (uniform over the workgroup; keys behind klen get zeros)
    const int chunks = p.D / X::E::CE, nqt = (p.Tq + X::KT - 1) / X::KT, n = G * nqt;
    const T* qb = reinterpret_cast<const T*>(p.q) + (long long)b * p.q_sb + (long long)hkv * G * p.q_sh;
    const T* gb = reinterpret_cast<const T*>(p.dout) + (long long)b * p.g_sb + (long long)hkv * G * p.g_sh;
    const long long srow = ((long long)b * p.H + (long long)hkv * G) * p.Tq;
    const int pitch = (p.Tq + 63) / 64 * 64;
    const long long nrow = (long long)p.B * p.H * pitch;
    const float* rows = p.rows + min(wave, 2) * nrow + ((long long)b * p.H + (long long)hkv * G) * pitch;
    unsigned ta[4];
    f32x4 none[NK];
    if constexpr (sizeof(T) == 2) x_tr_addr<DP>(ta, lds, r, g);
    XSource<T, DP> qs, gs;
    qs.init(qb, p.q_st, chunks, wave, lane);
    gs.init(gb, p.g_st, chunks, wave, lane);
    auto fetch = [&](int buf, int it) {
      const int hq = it / nqt, row0 = (it % nqt) * X::KT;
      // (scores of the rows behind the last query are taken from -inf; 0 as their query would be NaN against a key of -inf)
      qs.template request<true>(lds + buf * PAIR, (long long)hq * p.q_sh * (long long)sizeof(T), row0, p.Tq);
      gs.template request<false>(lds + buf * PAIR + X::BYTES, (long long)hq * p.g_sh * (long long)sizeof(T), row0, p.Tq);
      if (wave < 3)      // one of the three per wave
        __builtin_amdgcn_global_load_lds((x_glb_void*)(rows + (long long)hq * pitch + min(row0 + lane, pitch - 1)),
                                         (x_lds_void*)(lds + ROWS + buf * 1024 + wave * 256), 4, 0, 0);
    };
    fetch(0, 0);
    typename X::E::chunk K[NK][X::NS], V[NK][X::NS];
    x_load_rows<T, NK>(K, reinterpret_cast<const T*>(p.k) + (long long)b * p.k_sb + (long long)hkv * p.k_sh, p.k_st, k0, klen,
                          p.D, r, g);
    x_load_rows<T, NK>(V, reinterpret_cast<const T*>(p.v) + (long long)b * p.v_sb + (long long)hkv * p.v_sh, p.v_st, k0, klen,
                          p.D, r, g);
    x_turn<0>(true);
    auto step = [&](int it, auto BUF) {
      constexpr int BN = decltype(BUF)::value, AT = BN * PAIR;
      const float* sc = reinterpret_cast<const float*>(lds + ROWS + BN * 1024);
      if (it + 1 < n) fetch(1 - BN, it + 1);      // (that buffer was last read in step it - 1, behind that step's barrier)
      auto rows32 = [&](auto UC) {
        constexpr int u = decltype(UC)::value, R = AT + u * X::HALF;
        f32x4 s[NK][2], dp[NK][2];
        x_product<T, DP, NK>(s, lds + R, K, r, g, XZero());
        x_product<T, DP, NK>(dp, lds + R + X::BYTES, V, r, g, [&](int, int qf) -> f32x4 {
          return DROP ? f32x4{0.f, 0.f, 0.f, 0.f} : -*reinterpret_cast<const f32x4*>(sc + 128 + 32 * u + 16 * qf + 4 * g);
        });
        __builtin_amdgcn_sched_barrier(0);
        XAcross<T, DP> go, qo;
        XAcross<T, DP>::template read2<R + X::BYTES, R>(go, qo, lds, ta);
        __builtin_amdgcn_sched_barrier(0);
        if (uniform) {
#pragma unroll
          for (int f = 0; f < NK; ++f) s[f][0] = s[f][1] = f32x4{0.f, 0.f, 0.f, 0.f};      // (exponent 0 - 0, see the forward kernel)
        }
#pragma unroll
        for (int qf = 0; qf < 2; ++qf) {
          const int at = 32 * u + 16 * qf + 4 * g;
          const f32x4 m4 = *reinterpret_cast<const f32x4*>(sc + at);
          const f32x4 i4 = *reinterpret_cast<const f32x4*>(sc + 64 + at);
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(sc + 128 + at);
#pragma unroll
          for (int f = 0; f < NK; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = __builtin_amdgcn_exp2f(fmaf(s[f][qf][e], p.sl2, -m4[e]));
              if constexpr (sizeof(T) == 4) x *= i4[e];
              if constexpr (DROP) {
                const int qi = min((it % nqt) * X::KT + at + e, p.Tq - 1);
                const float keep = nsp_keep_scale(
                    p.seed, p.offset + (unsigned long long)((srow + (long long)(it / nqt) * p.Tq + qi) * p.Tk + k0 + 16 * f + r), p.drop);
                dp[f][qf][e] = x * fmaf(dp[f][qf][e], keep, -d4[e]);
                s[f][qf][e] = x * keep;
              } else {
                dp[f][qf][e] *= x;
                s[f][qf][e] = x;
              }
            }
        }
        go.template product<R + X::BYTES, false, NK>(dv, none, s, lds, r, g);
        qo.template product<R, false, NK>(dk, none, dp, lds, r, g);
      };
      rows32(std::integral_constant<int, 0>());
      if constexpr (X::U == 2) rows32(std::integral_constant<int, 1>());
      x_turn<0>(true);
    };
    for (int it = 0; it < n; it += 2) {
      step(it, std::integral_constant<int, 0>());
      if (it + 1 < n) step(it + 1, std::integral_constant<int, 1>());
    }
  }
#pragma unroll
  for (int f = 0; f < NK; ++f) {
    const int key = k0 + 16 * f + r;
    if (key >= p.Tk) continue;
    const long long at = (((long long)b * p.Tk + key) * p.Hkv + hkv) * p.D;
    if (key >= klen) {
#pragma unroll
      for (int i = 0; i < X::NB; ++i) dk[f][i] = dv[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (uniform) {      // the scores of such a row are constants
#pragma unroll
      for (int i = 0; i < X::NB; ++i) dk[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    x_store<DP>(reinterpret_cast<T*>(p.dk) + at, dk[f], p.scale, p.D, g);
    x_store<DP>(reinterpret_cast<T*>(p.dv) + at, dv[f], 1.f, p.D, g);
  }
}

template <typename T, int DP, int NQ, bool DROP>
int launch_fwd(const XArgs& p, hipStream_t st) {
  const long long per = (long long)(p.H / p.Hkv) * ((p.Tq + 64 * NQ - 1) / (64 * NQ));
  const long long wgs = ((long long)p.B * p.Hkv + 7) / 8 * 8 * per;
  if (wgs > 0x7fffffffLL) return NSP_EUNSUPPORTED;
  hipLaunchKernelGGL((cross_fwd_kernel<T, DP, NQ, DROP>), dim3((unsigned)wgs), dim3(256), 0, st, p);
  NSP_LAUNCH_CHECK();
  return NSP_OK;
}
template <typename T, int DP, bool DROP>
int launch_dq(const XArgs& p, hipStream_t st) {
  const long long wgs = ((long long)p.B * p.Hkv + 7) / 8 * 8 * (p.H / p.Hkv) * ((p.Tq + 63) / 64);
  if (wgs > 0x7fffffffLL) return NSP_EUNSUPPORTED;
  hipLaunchKernelGGL((cross_dq_kernel<T, DP, DROP>), dim3((unsigned)wgs), dim3(256), 0, st, p);
  NSP_LAUNCH_CHECK();
  return NSP_OK;
}
template <typename T, int DP, bool DROP>
int launch_dkv(const XArgs& p, hipStream_t st) {
  const long long wgs = ((long long)p.B * p.Hkv + 7) / 8 * 8 * ((p.Tk + 63) / 64);
  if (wgs > 0x7fffffffLL) return NSP_EUNSUPPORTED;
  hipLaunchKernelGGL((cross_dkv_kernel<T, DP, DROP>), dim3((unsigned)wgs), dim3(256), 0, st, p);
  NSP_LAUNCH_CHECK();
  return NSP_OK;
}

// Two owned 16-row fragments per wave halve the tile reads per score.  In the forward kernel they pay once the halved number of
// workgroups still fills the 256 compute units twice (bf16, 128 x 8 heads, 256 x 800, d 64: 104 -> 85 us; 32 x 16 heads, d 128:
// 113 -> 87; 4 x 16 heads, 500 x 2048, d 128, 256 workgroups left: 52 -> 61) and while there is no dropout, whose hashes then
// spill registers (the same calls: 184 -> 236 and 137 -> 187).  fp32 spends eight times as long in the matrix cores and keeps
// one.  So do dQ and dK / dV, whose accumulators leave too few registers for a third workgroup per compute unit (134 against 132
// and 205 against 205 us for the first of those calls; dK / dV 9.0 against 10.9 us for 32 x 8 heads, 61 x 90..187).
template <typename T, int DP, bool DROP>
int launch(const XArgs& p, bool bwd, hipStream_t st) {
  if (bwd) {
    const int rc = launch_dq<T, DP, DROP>(p, st);
    return rc != NSP_OK ? rc : launch_dkv<T, DP, DROP>(p, st);
  }
  if constexpr (sizeof(T) == 2 && !DROP)
    if (p.Tq > 64 && (long long)p.B * p.H * ((p.Tq + 127) / 128) >= 512) return launch_fwd<T, DP, 2, DROP>(p, st);
  return launch_fwd<T, DP, 1, DROP>(p, st);
}
template <typename T, bool DROP>
int launch_d(const XArgs& p, bool bwd, hipStream_t st) {
  if (p.D <= 32) return launch<T, 32, DROP>(p, bwd, st);
  if (p.D <= 64) return launch<T, 64, DROP>(p, bwd, st);
  return launch<T, 128, DROP>(p, bwd, st);
}

int cross_attn(const nsp_cross_attn_params* a, bool bwd, void* stream) {
  if (!a || a->B < 0 || a->Tq < 0 || a->Tk < 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->D <= 0) return NSP_EINVAL;
  if (a->D % 8 || a->D > 128 || (a->dtype != NSP_DT_F32 && a->dtype != NSP_DT_BF16)) return NSP_EUNSUPPORTED;
  if (a->B * a->H > 0x7ffffff0LL || a->Tq > 0x7fffff00LL || a->Tk > 0x7fffff00LL || !(a->scale > 0.)) return NSP_EUNSUPPORTED;
  // (32-bit offsets inside a tile; the stride of one row is never used and may be anything)
  const long long far = 1 << 24, q_st = a->Tq > 1 ? a->q_st : 0, k_st = a->Tk > 1 ? a->k_st : 0, v_st = a->Tk > 1 ? a->v_st : 0,
                  g_st = a->Tq > 1 ? a->g_st : 0;
  for (const long long ld : {q_st, k_st, v_st, g_st})
    if (ld < 0 || ld >= far) return NSP_EUNSUPPORTED;
  if (!(a->dropout_p >= 0. && a->dropout_p < 1.)) return NSP_EINVAL;
  if (a->B == 0 || a->Tk == 0 || a->Tq == 0) return NSP_OK;     // (no query or no key: zeros, which are the caller's)
  if (!a->q || !a->k || !a->v || !a->out) return NSP_EINVAL;
  if (bwd && (!a->dout || !a->dq || !a->dk || !a->dv || !a->stats || !a->rows)) return NSP_EINVAL;
  XArgs p;
  p.q = a->q; p.k = a->k; p.v = a->v; p.dout = a->dout; p.out = a->out;
  p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.stats = a->stats; p.rows = a->rows; p.klens = a->klens;
  p.B = (int)a->B; p.H = (int)a->H; p.Hkv = (int)a->Hkv; p.D = (int)a->D; p.Tq = (int)a->Tq; p.Tk = (int)a->Tk;
  p.q_sb = a->q_sb; p.q_st = q_st; p.q_sh = a->q_sh;
  p.k_sb = a->k_sb; p.k_st = k_st; p.k_sh = a->k_sh;
  p.v_sb = a->v_sb; p.v_st = v_st; p.v_sh = a->v_sh;
  p.g_sb = a->g_sb; p.g_st = g_st; p.g_sh = a->g_sh;
  p.seed = a->seed; p.offset = a->offset;
  p.scale = (float)a->scale;
  p.sl2 = (float)(a->scale * 1.4426950408889634);
  p.drop = (float)a->dropout_p;
  const hipStream_t st = (hipStream_t)stream;
  if (p.drop > 0.f)
    return a->dtype == NSP_DT_BF16 ? launch_d<__bf16, true>(p, bwd, st) : launch_d<float, true>(p, bwd, st);
  return a->dtype == NSP_DT_BF16 ? launch_d<__bf16, false>(p, bwd, st) : launch_d<float, false>(p, bwd, st);
}

}  // namespace

extern "C" int nsp_cross_attn_fwd(const nsp_cross_attn_params* a, void* stream) { return cross_attn(a, false, stream); }
extern "C" int nsp_cross_attn_bwd(const nsp_cross_attn_params* a, void* stream) { return cross_attn(a, true, stream); }
