// sample.hip -- one token per row of logits from given random numbers (temperature, top-k, top-p, min-p).
//
// Entries are ordered by falling logit, the lower index first among equals.  With w_i = exp((x_i - x_max) / T) kept are
//   the first k entries (top-k), of these the ones whose mass BEFORE them is below top_p x the mass of all k (so the entry that
//   completes top_p is the last), and of these the ones with w_i >= min_p;
// each rule keeps a prefix of the order and the first entry always stays.  The token is the first kept INDEX whose mass together
// with all kept indices before it exceeds u x the kept mass.
//
// A token is a whole number, so a sum that depends on the order of its additions, or a border that 32 bits blur, is a wrong
// answer now and then.  Masses are therefore fixed-point integers, w x 2^44 from a 64-bit exponential: integer sums have no
// order, and borders move by less than 2^-44 of the largest mass per entry.
//
// One workgroup per row: 4 waves for rows of up to 1024 logits, where latency is all, else 8.  A row is read once and stays in
// LDS, up to 10800 logits with their masses, so that the 64-bit exponential runs once per entry; rows behind 30000 logits
// are read again by each pass (from L2).  The k-th entry and the entry that completes top_p are found with one histogram
// whose bins are linear in the logit between the row's extremes, a scan, and an exact ranking of the few entries of the bin
// that the border falls in; rows with too many entries in that bin (equal logits) take a radix descent over (logit, index).
// Whatever can still be kept then goes to a list, if it is not too much for two entries per thread, and the remaining steps
// work on that instead of the row (256 rows of 10000 logits, top-k 500, top-p 0.9: 23.2 -> 14.7 us).
// What bounds the call is latency: about a dozen barriers, and scans over a wave, which therefore run on DPP lane moves
// (a step takes a few cycles, where a shuffle through LDS takes about 130), and the issue of what every wave has to do.
#include "common.h"

namespace {

typedef unsigned long long u64;
constexpr int CAND = 256;     // entries that are ranked one against the other
constexpr int FRAC = 44;      // bits behind the point of a mass; V <= 2^18 keeps every sum below 2^62
// what of the row the LDS holds
enum { NOTHING = 0, LOGITS = 1, LOGITS_AND_MASSES = 2 };

struct SampleArgs {
  const void* x;
  const float* u;
  const float* t;
  const int* k;
  const float* tp;
  const float* mp;
  int* out;
  long long ld;
  int V;
  int k_all;
  float t_all, tp_all, mp_all;
};

// four consecutive logits at any address (the memory system takes unaligned vectors)
typedef __attribute__((ext_vector_type(4), aligned(4))) float f32x4_any;
typedef __attribute__((ext_vector_type(4), aligned(2))) unsigned short u16x4_any;
__device__ __forceinline__ void sample_load4(const float* p, float (&y)[4]) {
  const f32x4_any v = *reinterpret_cast<const f32x4_any*>(p);
  y[0] = v[0]; y[1] = v[1]; y[2] = v[2]; y[3] = v[3];
}
__device__ __forceinline__ void sample_load4(const __bf16* p, float (&y)[4]) {
  const u16x4_any v = *reinterpret_cast<const u16x4_any*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = __uint_as_float((unsigned)v[j] << 16);
}

// order-preserving image of a logit (-0 counts as 0, a NaN as -inf), and of an entry: larger = earlier
__device__ __forceinline__ unsigned sample_key(float x) {
  if (x != x) return 0x007FFFFFu;
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float sample_logit(unsigned key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr int IDX_BITS = 20;
__device__ __forceinline__ u64 sample_entry(float x, int i) {
  return ((u64)sample_key(x) << IDX_BITS) | (u64)((1 << IDX_BITS) - 1 - i);
}

struct RowScale {
  float xmax;
  double inv_t;
  float bin_scale;
  // the histogram bin of a logit: it never falls as the logit falls, rounding included; -inf and NaN are in the last
  template <int BINS>
  __device__ __forceinline__ int bin(float x) const {
    const float z = (xmax - x) * bin_scale;
    return z < (float)(BINS - 1) ? (int)z : BINS - 1;
  }
};
// The mass of a logit: exp(d) x 2^44 rounded to a whole number, d = (x - xmax) / T <= 0; relative error of the exponential below
// 2^-47.  exp(d) = 2^n exp(f), |f| <= ln 2 / 2 (f = d - n ln 2 with ln 2 in two parts: Cody and Waite's reduction), the Taylor
// polynomial of the 11th degree; n and the final rounding come from additions of
// 1.5 x 2^52 and 2^52, whose low bits then are the whole number (gfx950 has no conversion from 64-bit floats to 64-bit integers).
__device__ __forceinline__ u64 sample_mass(float x, const RowScale& r) {
  const double d = x == r.xmax ? 0. : ((double)x - (double)r.xmax) * r.inv_t;
  const double t = fma(d, 1.4426950408889634074, 6755399441055744.0);
  const double n = t - 6755399441055744.0;
  const double f = fma(n, -2.3190468138462995584e-17, fma(n, -0.69314718055994528623, d));
  double s = 1.0 / 39916800.0;
  s = fma(s, f, 1.0 / 3628800.0);
  s = fma(s, f, 1.0 / 362880.0);
  s = fma(s, f, 1.0 / 40320.0);
  s = fma(s, f, 1.0 / 5040.0);
  s = fma(s, f, 1.0 / 720.0);
  s = fma(s, f, 1.0 / 120.0);
  s = fma(s, f, 1.0 / 24.0);
  s = fma(s, f, 1.0 / 6.0);
  s = fma(s, f, 0.5);
  s = fma(s, f, 1.0);
  s = fma(s, f, 1.0);
  const int e = (int)(unsigned)__builtin_bit_cast(u64, t);         // n
  const double scale = __builtin_bit_cast(double, (u64)(unsigned)(e + FRAC + 1023) << 52);
  const u64 m = __builtin_bit_cast(u64, fma(s, scale, 4503599627370496.0)) & ((1ull << 52) - 1);
  return d > -40.0 ? m : 0ull;       // (below 2^-57: no mass; also a NaN)
}

struct Mass4 {
  u64 m[4];
};
__device__ __forceinline__ Mass4 sample_mass4(float a, float b, float c, float d, const RowScale& rs) {
  return Mass4{{sample_mass(a, rs), sample_mass(b, rs), sample_mass(c, rs), sample_mass(d, rs)}};
}
// (for kernels that compute masses in several places: one copy of the code, everything in registers)
__device__ __attribute__((noinline)) Mass4 sample_mass4_call(float a, float b, float c, float d, float xmax, double inv_t) {
  return sample_mass4(a, b, c, d, RowScale{xmax, inv_t, 0.f});
}

// the value `CTRL` lanes below (DPP), 0 where there is none
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 lane_move(u64 v) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xF, true);
  return ((u64)(unsigned)hi << 32) | (unsigned)lo;
}
enum { ROW_SHR = 0x110, ROW_BCAST15 = 0x142, ROW_BCAST31 = 0x143 };
// sum over this lane and the ones below; lane 63 has the wave's
__device__ __forceinline__ u64 wave_scan(u64 v) {
  v += lane_move<ROW_SHR + 1, 0xF>(v);
  v += lane_move<ROW_SHR + 2, 0xF>(v);
  v += lane_move<ROW_SHR + 4, 0xF>(v);
  v += lane_move<ROW_SHR + 8, 0xF>(v);
  v += lane_move<ROW_BCAST15, 0xA>(v);
  v += lane_move<ROW_BCAST31, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 max_u64(u64 a, u64 b) { return a > b ? a : b; }
// maximum, in lane 63
__device__ __forceinline__ u64 wave_max(u64 v) {
  v = max_u64(v, lane_move<ROW_SHR + 1, 0xF>(v));
  v = max_u64(v, lane_move<ROW_SHR + 2, 0xF>(v));
  v = max_u64(v, lane_move<ROW_SHR + 4, 0xF>(v));
  v = max_u64(v, lane_move<ROW_SHR + 8, 0xF>(v));
  v = max_u64(v, lane_move<ROW_BCAST15, 0xA>(v));
  v = max_u64(v, lane_move<ROW_BCAST31, 0xC>(v));
  return v;
}

// the row's entries: thread t holds indices 4 ST c + 4 t + j of chunk c.  A thread reads back from LDS only what it wrote.
template <typename T, int ST, int KEEP>
struct Row {
  const T* p;
  f32x4* buf;        // [chunks][ST]
  ulonglong2* mbuf;  // [chunks][ST][2]
  RowScale rs;
  int V, chunks, tid;
  __device__ __forceinline__ void load(int c, float (&y)[4]) const {      // (indices behind the row: anything)
    const int i0 = c * (4 * ST) + 4 * tid;
    if (i0 + 3 < V) {
      sample_load4(p + i0, y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = i0 + j < V ? (float)p[i0 + j] : 0.f;
    }
  }
  __device__ __forceinline__ void get(int c, float (&y)[4]) const {
    if constexpr (KEEP != NOTHING) {
      const f32x4 v = buf[c * ST + tid];
      y[0] = v[0]; y[1] = v[1]; y[2] = v[2]; y[3] = v[3];
    } else {
      load(c, y);
    }
  }
  // one logit of this thread's
  __device__ __forceinline__ float logit(int i) const {
    if constexpr (KEEP != NOTHING) return reinterpret_cast<const float*>(buf)[i];
    else return (float)p[i];
  }
  // masses of the entries that are not below `floor`, 0 for the others
  __device__ __forceinline__ void compute(const float (&y)[4], int i0, u64 floor, u64 (&m)[4]) const {
    bool in[4], any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      in[j] = i0 + j < V && sample_entry(y[j], i0 + j) >= floor;
      any = any || in[j];
      m[j] = 0;
    }
    if (any) {
      const Mass4 w = KEEP == LOGITS_AND_MASSES ? sample_mass4(y[0], y[1], y[2], y[3], rs)
                                                : sample_mass4_call(y[0], y[1], y[2], y[3], rs.xmax, rs.inv_t);
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = in[j] ? w.m[j] : 0;
    }
  }
  // LOGITS_AND_MASSES: the masses the later passes find in LDS
  __device__ __forceinline__ void keep_masses(u64 floor) {
    if constexpr (KEEP == LOGITS_AND_MASSES) {
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        const int i0 = c * (4 * ST) + 4 * tid;
        if (i0 >= V) break;
        float y[4];
        u64 m[4];
        get(c, y);
        compute(y, i0, floor, m);
        mbuf[2 * (c * ST + tid)] = make_ulonglong2(m[0], m[1]);
        mbuf[2 * (c * ST + tid) + 1] = make_ulonglong2(m[2], m[3]);
      }
    }
  }
  // the masses again, for the floor of keep_masses or (RISEN) a higher one
  template <bool RISEN>
  __device__ __forceinline__ void masses(int c, const float (&y)[4], int i0, u64 floor, u64 (&m)[4]) const {
    if constexpr (KEEP == LOGITS_AND_MASSES) {
      const ulonglong2 a = mbuf[2 * (c * ST + tid)], b = mbuf[2 * (c * ST + tid) + 1];
      m[0] = a.x; m[1] = a.y; m[2] = b.x; m[3] = b.y;
      if constexpr (RISEN) {
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = sample_entry(y[j], i0 + j) < floor ? 0 : m[j];
      }
    } else {
      compute(y, i0, floor, m);
    }
  }
  // f(chunk, x[4], first index), for the chunks where this thread has an entry (WHOLE: for all, whole waves)
  template <bool WHOLE, int UNROLL, class F>
  __device__ __forceinline__ void each_chunk(F f) {
#pragma unroll UNROLL
    for (int c = 0; c < chunks; ++c) {
      const int i0 = c * (4 * ST) + 4 * tid;
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      if (i0 < V) get(c, y);
      else if (!WHOLE) continue;
      f(c, y, i0);
    }
  }
};

template <int ST>
struct Shared {
  u64 hist[3][2 * ST];   // counts per bin, masses per bin, masses per segment of the row
  u64 cand[CAND];        // entries of the border's bin
  u64 cmass[CAND];
  u64 red[4][16];        // (one for each use: no barrier in front of the next)
  u64 before[3], last[2];
  int bin[3], count[4], listed;
};

// sums over the waves below (off) and over all (all) from each wave's own, `to` in its lane 63; one barrier
template <int ST>
__device__ __forceinline__ void block_sums(u64* red, u64 to, int tid, u64& off, u64& all) {
  constexpr int NW = ST / 64;
  const int lane = tid & 63, wave = tid >> 6;
  if (lane == 63) red[wave] = to;
  __syncthreads();
  u64 s = lane < NW ? red[lane] : 0;
  s += lane_move<ROW_SHR + 1, 0xF>(s);
  s += lane_move<ROW_SHR + 2, 0xF>(s);
  if (NW > 4) s += lane_move<ROW_SHR + 4, 0xF>(s);
  all = __shfl(s, NW - 1, 64);
  off = __shfl(s, wave > 0 ? wave - 1 : 0, 64);
  if (wave == 0) off = 0;
}

// The bin (0 = the first of the order) that the border falls in: the last non-empty one with less than the border before it,
// where `base` is what lies before bin 0.  The border is `target` entries, or the mass `lim` (frac > 0: frac x the bins' whole).
// -> sh.bin[W], sh.before[W] (base included); returns lim
template <int ST, bool MASS>
__device__ __forceinline__ double find_bin(Shared<ST>& sh, u64 base, u64 target, double lim, double frac, int tid) {
  constexpr int W = MASS ? 1 : 0;
  const u64 a = sh.hist[W][2 * tid], b = sh.hist[W][2 * tid + 1];
  const u64 to = wave_scan(a + b);
  u64 off, all;
  block_sums<ST>(sh.red[W], to, tid, off, all);
  if (MASS && frac > 0.) lim = frac * (double)all;
  auto below = [&](u64 s) -> bool { return MASS ? (double)(base + s) < lim : base + s < target; };
  // sums before the bins rise: a kept bin is the last one if the sum behind it is not below the border, or is the whole
  const u64 s2 = off + to, s1 = s2 - b, s0 = s1 - a;
  if (b > 0 && below(s1) && (!below(s2) || s2 == all)) { sh.bin[W] = 2 * tid + 1; sh.before[W] = base + s1; }
  else if (a > 0 && below(s0) && (!below(s1) || s1 == all)) { sh.bin[W] = 2 * tid; sh.before[W] = base + s0; }
  __syncthreads();
  return lim;
}

// The last kept entry when all entries take part with weight 1 (count: the first `target` stay), or the ones >= floor with their
// mass (those with less than frac x the whole before them stay).  sh.hist[W], sh.count[W] and sh.last[W] come cleared.
// Entries up to the border's bin also go to the list, in any order: sh.listed of them in sh.hist[0], or more than it holds.
template <typename T, int ST, int KEEP, bool MASS>
__device__ __forceinline__ u64 last_kept(Shared<ST>& sh, Row<T, ST, KEEP>& row, u64 floor, u64 target, double frac) {
  constexpr int BINS = 2 * ST, LOG_BINS = ST == 512 ? 10 : 9, W = MASS ? 1 : 0;
  static_assert(BINS == 1 << LOG_BINS, "bins");
  const int tid = row.tid;
  auto each = [&](auto f) {       // f(x, index, weight, bin) for the entries that take part
    row.template each_chunk<false, MASS ? 1 : 4>([&](int c, float (&y)[4], int i0) {
      u64 m[4] = {1, 1, 1, 1};
      if constexpr (MASS) row.template masses<false>(c, y, i0, floor, m);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = row.rs.template bin<BINS>(y[j]);
        if (MASS ? m[j] > 0 : i0 + j < row.V) f(y[j], i0 + j, m[j], b);
      }
    });
  };
  each([&](float, int, u64 m, int b) { atomicAdd(&sh.hist[W][b], m); });
  __syncthreads();
  const double lim = find_bin<ST, MASS>(sh, 0, target, 0., frac, tid);
  const int bin = sh.bin[W];
  const u64 before = sh.before[W];
  // (count: their number is known; hist[0] is free from here on)
  const bool list = MASS || before + sh.hist[0][bin] <= (u64)BINS;
  __syncthreads();
  // Few entries are left: a pass marks them, 16 chunks at a time, and what is done per entry runs over the marks (a branch per
  // entry of the row took 4.1 us of 10000 logits, this 2.3).  On the list a thread's entries are side by side, the waves in any order.
  const bool last = bin == BINS - 1;
  const float reach = (float)(bin + 1);
#pragma unroll 1
  for (int c0 = 0; c0 < row.chunks; c0 += 16) {
    u64 marks = 0;
    const int c1 = min(c0 + 16, row.chunks);
#pragma unroll 4
    for (int c = c0; c < c1; ++c) {
      const int i0 = c * (4 * ST) + 4 * tid;
      if (i0 >= row.V) continue;
      float y[4];
      row.get(c, y);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bool in = i0 + j < row.V && (last || (row.rs.xmax - y[j]) * row.rs.bin_scale < reach);      // (rs.bin(y[j]) <= bin)
        if (MASS) in = in && sample_entry(y[j], i0 + j) >= floor;
        marks |= (u64)(in ? 1u << j : 0u) << (4 * (c - c0));
      }
    }
    int at = 0;
    if (list) {
      const int mine = __builtin_popcountll(marks), to = (int)wave_scan((u64)mine);
      int base = 0;
      if ((tid & 63) == 63) base = atomicAdd(&sh.count[2 + W], to);
      at = __shfl(base, 63, 64) + to - mine;
    }
    while (marks) {
      const int bit = __builtin_ctzll(marks), i = (c0 + (bit >> 2)) * (4 * ST) + 4 * tid + (bit & 3);
      marks &= marks - 1;
      const float x = row.logit(i);
      const u64 c = sample_entry(x, i);
      if (list && at < BINS) sh.hist[0][at] = c;
      ++at;
      if (row.rs.template bin<BINS>(x) == bin) {
        const u64 m = MASS ? sample_mass(x, row.rs) : 1;
        if (m > 0) {
          const int o = atomicAdd(&sh.count[W], 1);
          if (o < CAND) { sh.cand[o] = c; sh.cmass[o] = m; }
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.count[W];
  if (tid == 0) sh.listed = list && n <= CAND ? sh.count[2 + W] : BINS + 1;
  if (n <= CAND) {
    // rank every candidate against the others; the last kept one is the smallest entry with less than the border before it
    if (tid < n) {
      const u64 c = sh.cand[tid];
      u64 s = before;
#pragma unroll 4
      for (int o = 0; o < n; ++o) s += sh.cand[o] > c ? sh.cmass[o] : 0;
      if (MASS ? (double)s < lim : s < target) atomicMin(&sh.last[W], c);
    }
    __syncthreads();
    return sh.last[W];
  }
  // many equal logits: radix descent over the entries of the bin
  u64 prefix = 0, sum = before;
#pragma unroll 1
  for (int hi = 32 + IDX_BITS; hi > 0;) {
    const int bits = hi > LOG_BINS ? LOG_BINS : hi, lo = hi - bits;
    __syncthreads();
    sh.hist[W][2 * tid] = 0;
    sh.hist[W][2 * tid + 1] = 0;
    __syncthreads();
    each([&](float x, int i, u64 m, int b) {
      const u64 c = sample_entry(x, i);
      if (b == bin && (c >> hi) == prefix) atomicAdd(&sh.hist[W][(1 << bits) - 1 - (int)((c >> lo) & ((1u << bits) - 1u))], m);
    });
    __syncthreads();
    find_bin<ST, MASS>(sh, sum, target, lim, 0., tid);
    prefix = (prefix << bits) | (u64)((1 << bits) - 1 - sh.bin[W]);
    sum = sh.before[W];
    hi = lo;
  }
  __syncthreads();
  return prefix;
}

template <typename T, int ST, int KEEP>
__global__ __launch_bounds__(ST) void sample_rows_kernel(const SampleArgs a) {
  constexpr int NW = ST / 64;
  __shared__ Shared<ST> sh;
  extern __shared__ __attribute__((aligned(16))) float row_buf[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long b = blockIdx.x;
  Row<T, ST, KEEP> row;
  row.p = reinterpret_cast<const T*>(a.x) + b * a.ld;
  row.V = a.V;
  row.tid = tid;
  row.chunks = (a.V + 4 * ST - 1) / (4 * ST);
  row.buf = reinterpret_cast<f32x4*>(row_buf);
  row.mbuf = reinterpret_cast<ulonglong2*>(row_buf + (a.V + 3) / 4 * 4);
  const float t = a.t ? a.t[b] : a.t_all, tp = a.tp ? a.tp[b] : a.tp_all, mp = a.mp ? a.mp[b] : a.mp_all;
  const float u = a.u[b];
  int k = a.k ? a.k[b] : a.k_all;
  if (k <= 0 || k > a.V) k = a.V;

  // while the row is on its way
#pragma unroll
  for (int w = 0; w < 3; ++w) sh.hist[w][2 * tid] = sh.hist[w][2 * tid + 1] = 0;
  if (tid < 4) sh.count[tid] = 0;
  if (tid < 2) sh.last[tid] = ~0ull;
  if (tid == 4) sh.listed = 2 * ST + 1;

  // the row; the first entry of the order, and the smallest finite logit (as the largest complemented key)
  u64 top = 0, low = 0;
#pragma unroll 4
  for (int c = 0; c < row.chunks; ++c) {
    const int i0 = c * (4 * ST) + 4 * tid;
    if (i0 >= a.V) break;
    float y[4];
    row.load(c, y);
    if constexpr (KEEP != NOTHING) row.buf[c * ST + tid] = f32x4{y[0], y[1], y[2], y[3]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j < a.V) {
        top = max_u64(top, sample_entry(y[j], i0 + j));
        if (y[j] > -INFINITY) low = max_u64(low, (u64)(unsigned)~sample_key(y[j]));
      }
    }
  }
  top = wave_max(top);
  low = wave_max(low);
  if (lane == 63) { sh.red[2][wave] = top; sh.red[3][wave] = low; }
  __syncthreads();
  top = low = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    top = max_u64(top, sh.red[2][w]);
    low = max_u64(low, sh.red[3][w]);
  }
  const int first = (1 << IDX_BITS) - 1 - (int)(top & ((1u << IDX_BITS) - 1u));
  const unsigned tk = (unsigned)(top >> IDX_BITS), lk = ~(unsigned)low;
  row.rs.xmax = sample_logit(tk);
  const float xmin = sample_logit(lk);
  // temperature 0, one entry, nothing but -inf / NaN: the first entry
  if (!(t > 0.f) || k == 1 || !(tp > 0.f) || tk <= 0x007FFFFFu) {
    if (tid == 0) a.out[b] = first;
    return;
  }
  row.rs.inv_t = 1.0 / (double)t;
  const float range = row.rs.xmax - xmin;
  row.rs.bin_scale = range > 0.f && range < INFINITY ? (float)(2 * ST - 1) / range : 0.f;

  // min_p as a mass (NaN: all but the first out)
  const double least = ceil((double)mp * (double)(1ull << FRAC));
  const u64 min_mass = least <= 0. ? 0ull : least < 9e15 ? (u64)least : ~0ull;
  auto inside = [](u64 from, u64 m, u64 all, double want) -> bool {      // does the token's point fall into [from, from + m)
    return m > 0 && (!((double)from > want) || from == 0) && ((double)(from + m) > want || from + m == all);
  };

  u64 floor = 0;
  const bool by_count = k < a.V;
  if (by_count) floor = last_kept<T, ST, KEEP, false>(sh, row, 0, (u64)k, 0.);
  bool by_mass = tp < 1.f;
  if (!by_count || sh.listed > 2 * ST) {
    row.keep_masses(floor);
    if (by_mass) floor = last_kept<T, ST, KEEP, true>(sh, row, floor, 0, (double)tp);
    by_mass = false;
  }
  if (sh.listed <= 2 * ST) {
    // What can stay is on the list, two entries per thread: the rest of the work is on these, whatever the row's length.
    const int n = sh.listed;
    u64 c[2], m[2];
    int bin[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      c[j] = tid + j * ST < n ? sh.hist[0][tid + j * ST] : 0;
      const float x = sample_logit((unsigned)(c[j] >> IDX_BITS));
      m[j] = c[j] >= floor && c[j] > 0 ? sample_mass(x, row.rs) : 0;
      bin[j] = row.rs.template bin<2 * ST>(x);
    }
    if (by_mass) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (m[j]) atomicAdd(&sh.hist[1][bin[j]], m[j]);
      __syncthreads();
      const double lim = find_bin<ST, true>(sh, 0, 0, 0., (double)tp, tid);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        sh.hist[1][tid + j * ST] = m[j];      // (now beside hist[0]: the masses of the list)
        if (m[j] && bin[j] == sh.bin[1]) {
          const int at = atomicAdd(&sh.count[1], 1);
          if (at < CAND) { sh.cand[at] = c[j]; sh.cmass[at] = m[j]; }
        }
      }
      __syncthreads();
      const int nc = sh.count[1];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (m[j] && bin[j] == sh.bin[1]) {
          u64 s = 0;
          if (nc <= CAND) {
            s = sh.before[1];
#pragma unroll 4
            for (int o = 0; o < nc; ++o) s += sh.cand[o] > c[j] ? sh.cmass[o] : 0;
          } else {      // more equal logits than candidates: over the whole list
            for (int o = 0; o < n; ++o) s += sh.hist[0][o] > c[j] ? sh.hist[1][o] : 0;
          }
          if ((double)s < lim) atomicMin(&sh.last[1], c[j]);
        }
      __syncthreads();
      floor = sh.last[1];
    }
    // the kept mass by index: bins of 2^shift indices, then the entries of the bin that the point falls in
    int shift = 0;
    while ((a.V - 1) >> shift >= 2 * ST) ++shift;
    int idx[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      idx[j] = (1 << IDX_BITS) - 1 - (int)(c[j] & ((1u << IDX_BITS) - 1u));
      if (c[j] < floor || !(m[j] >= min_mass || idx[j] == first)) m[j] = 0;
      if (m[j]) atomicAdd(&sh.hist[2][idx[j] >> shift], m[j]);
    }
    if (tid == 0) sh.count[0] = 0;
    __syncthreads();
    const u64 ha = sh.hist[2][2 * tid], hb = sh.hist[2][2 * tid + 1];
    const u64 to = wave_scan(ha + hb);
    u64 off, all;
    block_sums<ST>(sh.red[2], to, tid, off, all);
    const double want = (double)u * (double)all;
    const u64 end = off + to;
    if (inside(end - hb - ha, ha, all, want)) { sh.bin[2] = 2 * tid; sh.before[2] = end - hb - ha; }
    if (inside(end - hb, hb, all, want)) { sh.bin[2] = 2 * tid + 1; sh.before[2] = end - hb; }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (m[j] && idx[j] >> shift == sh.bin[2]) {
        const int at = atomicAdd(&sh.count[0], 1);      // (at most 2^shift <= 256 = CAND of them)
        sh.cand[at] = (u64)idx[j];
        sh.cmass[at] = m[j];
      }
    __syncthreads();
    if (tid < sh.count[0]) {
      const u64 i = sh.cand[tid];
      u64 s = sh.before[2];
      for (int o = 0; o < sh.count[0]; ++o) s += sh.cand[o] < i ? sh.cmass[o] : 0;
      if (inside(s, sh.cmass[tid], all, want)) a.out[b] = (int)i;
    }
    return;
  }

  // kept mass by index: per chunk and wave (256 consecutive indices), in sh.hist[2]
  auto kept_masses = [&](int c, float (&y)[4], int i0, u64 (&m)[4]) {
    m[0] = m[1] = m[2] = m[3] = 0;
    if (i0 >= a.V) return;
    row.template masses<true>(c, y, i0, floor, m);
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = m[j] >= min_mass || i0 + j == first ? m[j] : 0;
  };
  row.template each_chunk<true, 1>([&](int c, float (&y)[4], int i0) {
    u64 m[4];
    kept_masses(c, y, i0, m);
    const u64 s = wave_scan(m[0] + m[1] + m[2] + m[3]);
    if (lane == 63) sh.hist[2][c * NW + wave] = s;
  });
  __syncthreads();
  // the segment of the token: the first whose end exceeds u x the whole (u >= 1, NaN: the last with any mass)
  const u64 ha = sh.hist[2][2 * tid], hb = sh.hist[2][2 * tid + 1];
  const u64 to = wave_scan(ha + hb);
  u64 off, all;
  block_sums<ST>(sh.red[2], to, tid, off, all);
  const double want = (double)u * (double)all;
  const u64 end = off + to;
  if (inside(end - hb - ha, ha, all, want)) { sh.bin[2] = 2 * tid; sh.before[2] = end - hb - ha; }
  if (inside(end - hb, hb, all, want)) { sh.bin[2] = 2 * tid + 1; sh.before[2] = end - hb; }
  __syncthreads();
  const int seg = sh.bin[2];
  if (wave != seg % NW) return;
  const int c = seg / NW, i0 = c * (4 * ST) + 4 * tid;
  float y[4] = {0.f, 0.f, 0.f, 0.f};
  u64 m[4];
  if (i0 < a.V) row.get(c, y);
  kept_masses(c, y, i0, m);
  const u64 s = m[0] + m[1] + m[2] + m[3];
  u64 at = sh.before[2] + wave_scan(s) - s;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (inside(at, m[j], all, want)) a.out[b] = i0 + j;
    at += m[j];
  }
}

template <typename T, int ST, int KEEP>
int launch_sample(const SampleArgs& a, long long rows, hipStream_t st) {
  const size_t v4 = ((size_t)a.V + 3) / 4 * 4, bytes = KEEP == NOTHING ? 0 : KEEP == LOGITS ? v4 * 4 : v4 * 12;
  if (bytes + sizeof(Shared<ST>) > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)sample_rows_kernel<T, ST, KEEP>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 130000);
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL((sample_rows_kernel<T, ST, KEEP>), dim3((unsigned)rows), dim3(ST), bytes, st, a);
  NSP_LAUNCH_CHECK();
  return NSP_OK;
}
template <typename T>
int launch_sample_v(const SampleArgs& a, long long rows, hipStream_t st) {
  if (a.V <= 1024) return launch_sample<T, 256, LOGITS_AND_MASSES>(a, rows, st);
  if (a.V <= 10800) return launch_sample<T, 512, LOGITS_AND_MASSES>(a, rows, st);   // 127 KB beside the 29 KB of Shared
  if (a.V <= 30000) return launch_sample<T, 512, LOGITS>(a, rows, st);
  return launch_sample<T, 512, NOTHING>(a, rows, st);
}

}  // namespace

extern "C" int nsp_sample_rows(const nsp_sample_params* s, void* stream) {
  if (!s || s->rows < 0 || s->V <= 0) return NSP_EINVAL;
  if (s->rows == 0) return NSP_OK;
  if (!s->x || !s->u || !s->out || s->ld < s->V) return NSP_EINVAL;
  if (s->V > (1 << 18) || s->rows > 0x7fffffffLL) return NSP_EUNSUPPORTED;
  SampleArgs a;
  a.x = s->x; a.u = s->u; a.t = s->temperature; a.k = s->top_k; a.tp = s->top_p; a.mp = s->min_p; a.out = s->out;
  a.ld = s->ld;
  a.V = (int)s->V;
  a.k_all = s->k_all > 0x7fffffffLL ? 0x7fffffff : (int)(s->k_all < 0 ? 0 : s->k_all);
  a.t_all = (float)s->t_all; a.tp_all = (float)s->tp_all; a.mp_all = (float)s->mp_all;
  if (s->dtype == NSP_DT_F32) return launch_sample_v<float>(a, s->rows, (hipStream_t)stream);
  if (s->dtype == NSP_DT_BF16) return launch_sample_v<__bf16>(a, s->rows, (hipStream_t)stream);
  return NSP_EUNSUPPORTED;
}
