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
// One workgroup of 16 waves per row.  A row of up to 32768 logits is read once and stays in LDS, a longer one is read again
// by each pass (from L2).  The k-th entry and the entry that completes top_p are found with one histogram of 2048
// bins that are linear in the logit between the row's extremes, a scan, and an exact ranking of the few entries of the bin
// that the border falls in; rows with too many entries in that bin (equal logits) take a radix descent over (logit, index).
// What bounds the call is latency: a handful of workgroup-wide reductions of about half a microsecond each.
#include "common.h"

namespace {

typedef unsigned long long u64;
constexpr int ST = 1024;      // threads
constexpr int NW = ST / 64;   // waves
constexpr int BINS = 2048;
constexpr int ROW_CHUNKS = 8; // chunks of 4096 logits that fit the LDS (128 KB) beside `Shared`
constexpr int CAND = 512;    // entries that are ranked one against the other
constexpr int FRAC = 44;      // bits behind the point of a mass; V <= 2^18 keeps every sum below 2^62

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

__device__ __forceinline__ float sample_load(const float* p) { return *p; }
__device__ __forceinline__ float sample_load(const __bf16* p) { return (float)*p; }

// order-preserving image of a logit (-0 counts as 0; a NaN is below everything), and of an entry: larger = earlier
__device__ __forceinline__ unsigned sample_key(float x) {
  if (x != x) return 0u;
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
constexpr int IDX_BITS = 20;
__device__ __forceinline__ u64 sample_entry(float x, int i) {
  return ((u64)sample_key(x) << IDX_BITS) | (u64)((1 << IDX_BITS) - 1 - i);
}

// exp(d), d <= 0, to better than 2^-46 of its value: exp(d) = 2^n exp(f), |f| <= ln 2 / 2, Taylor to the 12th power
__device__ __forceinline__ double sample_exp(double d) {
  const double n = rint(d * 1.4426950408889634074);
  const double f = fma(n, -2.3190468138462995584e-17, fma(n, -0.69314718055994528623, d));
  double s = 1.0 / 479001600.0;
  s = fma(s, f, 1.0 / 39916800.0);
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
  return ldexp(s, (int)n);
}

struct RowScale {
  float xmax;
  double inv_t;
};
__device__ __forceinline__ double sample_weight(float x, const RowScale& r) {
  if (x == r.xmax) return 1.0;
  const double d = ((double)x - (double)r.xmax) * r.inv_t;
  return d > -40.0 ? sample_exp(d) : 0.0;       // (below 2^-57: no mass; also a NaN)
}
__device__ __forceinline__ u64 sample_mass(double w) { return (u64)(w * (double)(1ull << FRAC) + 0.5); }

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 w = __shfl_xor(v, o, 64);
    v = w > v ? w : v;
  }
  return v;
}
// sum over the lanes below
__device__ __forceinline__ u64 wave_before_u64(u64 v, int lane) {
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 w = __shfl_up(s, o, 64);
    if (lane >= o) s += w;
  }
  return s - v;
}

// the row's entries: thread t holds indices 4 ST c + 4 t + j of chunk c.  IN_LDS: read once, kept in LDS
template <typename T, bool IN_LDS>
struct Row {
  const T* p;
  f32x4* buf;
  int V, chunks, tid;
  __device__ __forceinline__ void fetch(int c, float (&y)[4]) const {
    const int i0 = c * (4 * ST) + 4 * tid;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = i0 + j < V ? sample_load(p + i0 + j) : 0.f;
  }
  __device__ __forceinline__ void init() {
    if constexpr (IN_LDS) {      // (a thread reads back only what it wrote)
#pragma unroll 4
      for (int c = 0; c < chunks; ++c) {
        float y[4];
        fetch(c, y);
        buf[c * ST + tid] = f32x4{y[0], y[1], y[2], y[3]};
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void each_chunk(F f) {   // f(chunk, x[4], first index)
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      float y[4];
      if constexpr (IN_LDS) {
        const f32x4 v = buf[c * ST + tid];
        y[0] = v[0]; y[1] = v[1]; y[2] = v[2]; y[3] = v[3];
      } else {
        fetch(c, y);
      }
      f(c, y, c * (4 * ST) + 4 * tid);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) {         // f(x, index) for the entries that there are
    const int n = V;
    each_chunk([&](int, float (&y)[4], int i0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j < n) f(y[j], i0 + j);
    });
  }
};

struct Shared {
  u64 hist[BINS];     // counts or masses per bin
  u64 cand[CAND];     // entries of the border's bin
  u64 cmass[CAND];
  u64 red[NW], red2[NW];
  u64 before;
  int bin, count;
};

// The bin (0 = the first of the order) that the border falls in: the last non-empty one with less than the border before it,
// where `base` is what lies before bin 0.  The border is `target` entries, or the mass `lim` (frac > 0: frac x the bins' whole).
// -> sh.bin, sh.before (base included); returns lim
template <bool MASS>
__device__ __forceinline__ double find_bin(Shared& sh, u64 base, u64 target, double lim, double frac, int tid) {
  const int lane = tid & 63, wave = tid >> 6;
  const u64 a = sh.hist[2 * tid], b = sh.hist[2 * tid + 1];
  const u64 inw = wave_before_u64(a + b, lane);
  if (lane == 63) sh.red[wave] = inw + a + b;
  if (tid == 0) { sh.bin = 0; sh.before = base; }
  __syncthreads();
  u64 off = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const u64 s = sh.red[w];
    off += w < wave ? s : 0;
    all += s;
  }
  if (MASS && frac > 0.) lim = frac * (double)all;
  auto below = [&](u64 s) -> bool { return MASS ? (double)(base + s) < lim : base + s < target; };
  // sums before the bins rise: a kept bin is the last one if the sum behind it is not below the border, or is the whole
  const u64 s0 = off + inw, s1 = s0 + a, s2 = s1 + b;
  if (b > 0 && below(s1) && (!below(s2) || s2 == all)) { sh.bin = 2 * tid + 1; sh.before = base + s1; }
  else if (a > 0 && below(s0) && (!below(s1) || s1 == all)) { sh.bin = 2 * tid; sh.before = base + s0; }
  __syncthreads();
  return lim;
}

// The last kept entry when entries >= floor take part with weight 1 (count: the first `target` stay) or their mass (those
// with less than frac x the whole before them stay).
template <typename T, bool IN_LDS, bool MASS>
__device__ u64 last_kept(Shared& sh, Row<T, IN_LDS>& row, const RowScale& rs, u64 floor, float bin_scale, u64 target, double frac) {
  const int tid = row.tid;
  auto weight = [&](float x) -> u64 { return MASS ? sample_mass(sample_weight(x, rs)) : 1ull; };
  auto bin_of = [&](float x) -> int {
    const float y = (rs.xmax - x) * bin_scale;            // falls as x rises, rounding included
    return y < (float)(BINS - 1) ? (int)y : BINS - 1;      // (-inf, NaN: last)
  };
  __syncthreads();
  sh.hist[2 * tid] = 0;
  sh.hist[2 * tid + 1] = 0;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  row.each([&](float x, int i) {
    if (sample_entry(x, i) >= floor) {
      const u64 w = weight(x);
      if (w) atomicAdd(&sh.hist[bin_of(x)], w);
    }
  });
  __syncthreads();
  const double lim = find_bin<MASS>(sh, 0, target, 0., frac, tid);
  const int bin = sh.bin;
  const u64 before = sh.before;
  row.each([&](float x, int i) {
    if (bin_of(x) == bin && sample_entry(x, i) >= floor) {
      const u64 w = weight(x);
      if (w) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < CAND) { sh.cand[at] = sample_entry(x, i); sh.cmass[at] = w; }
      }
    }
  });
  __syncthreads();
  const int n = sh.count;
  if (n <= CAND) {
    // rank every candidate against the others; the last kept one is the smallest entry with less than the border before it
    u64 mine = ~0ull;
    for (int a = tid; a < n; a += ST) {
      const u64 c = sh.cand[a];
      u64 s = before;
      for (int o = 0; o < n; ++o) s += sh.cand[o] > c ? sh.cmass[o] : 0;
      if (MASS ? (double)s < lim : s < target) mine = c;
    }
    mine = ~wave_max_u64(~mine);
    if ((tid & 63) == 0) sh.red2[tid >> 6] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) mine = sh.red2[w] < mine ? sh.red2[w] : mine;
    return mine;
  }
  // many equal logits: radix descent over the entries of the bin, 11 bits at a time
  u64 prefix = 0, sum = before;
  for (int hi = 32 + IDX_BITS; hi > 0;) {
    const int bits = hi > 11 ? 11 : hi, lo = hi - bits;
    __syncthreads();
    sh.hist[2 * tid] = 0;
    sh.hist[2 * tid + 1] = 0;
    __syncthreads();
    row.each([&](float x, int i) {
      const u64 c = sample_entry(x, i);
      if (c >= floor && bin_of(x) == bin && (c >> hi) == prefix) {
        const u64 w = weight(x);
        if (w) atomicAdd(&sh.hist[(1 << bits) - 1 - (int)((c >> lo) & ((1u << bits) - 1u))], w);
      }
    });
    __syncthreads();
    find_bin<MASS>(sh, sum, target, lim, 0., tid);
    prefix = (prefix << bits) | (u64)((1 << bits) - 1 - sh.bin);
    sum = sh.before;
    hi = lo;
  }
  return prefix;
}

template <typename T, bool IN_LDS>
__global__ __launch_bounds__(ST) void sample_rows_kernel(const SampleArgs a) {
  __shared__ Shared sh;
  extern __shared__ __attribute__((aligned(16))) float row_buf[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long b = blockIdx.x;
  Row<T, IN_LDS> row;
  row.p = reinterpret_cast<const T*>(a.x) + b * a.ld;
  row.V = a.V;
  row.tid = tid;
  row.buf = reinterpret_cast<f32x4*>(row_buf);
  row.chunks = (a.V + 4 * ST - 1) / (4 * ST);
  const float t = a.t ? a.t[b] : a.t_all, tp = a.tp ? a.tp[b] : a.tp_all, mp = a.mp ? a.mp[b] : a.mp_all;
  const float u = a.u[b];
  int k = a.k ? a.k[b] : a.k_all;
  if (k <= 0 || k > a.V) k = a.V;
  row.init();

  // first entry of the order, and the smallest finite logit
  u64 top = 0;
  float mn = INFINITY;
  row.each([&](float x, int i) {
    const u64 c = sample_entry(x, i);
    top = c > top ? c : top;
    if (x > -INFINITY && x < mn) mn = x;
  });
  top = wave_max_u64(top);
  mn = -wave_reduce_max(-mn);
  if (lane == 0) { sh.red[wave] = top; sh.red2[wave] = __float_as_uint(mn); }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    top = sh.red[w] > top ? sh.red[w] : top;
    mn = fminf(mn, __uint_as_float((unsigned)sh.red2[w]));
  }
  const int first = (1 << IDX_BITS) - 1 - (int)(top & ((1u << IDX_BITS) - 1u));
  const unsigned tk = (unsigned)(top >> IDX_BITS);
  RowScale rs;
  rs.xmax = __uint_as_float(tk ^ ((tk >> 31) ? 0x80000000u : 0xFFFFFFFFu));
  // temperature 0, one entry, nothing but -inf / NaN: the first entry
  if (!(t > 0.f) || k == 1 || !(tp > 0.f) || tk <= 0x007FFFFFu) {
    if (tid == 0) a.out[b] = first;
    return;
  }
  rs.inv_t = 1.0 / (double)t;
  const float range = rs.xmax - mn;
  const float bin_scale = range > 0.f && range < INFINITY ? (float)(BINS - 1) / range : 0.f;

  u64 floor = 0;
  if (k < a.V) floor = last_kept<T, IN_LDS, false>(sh, row, rs, 0, bin_scale, (u64)k, 0.);
  if (tp < 1.f) floor = last_kept<T, IN_LDS, true>(sh, row, rs, floor, bin_scale, 0, (double)tp);

  // kept mass by index: per chunk and wave (256 consecutive indices), in sh.hist
  const double minw = (double)mp;
  auto mass = [&](float x, int i) -> u64 {
    const u64 c = sample_entry(x, i);
    if (c < floor) return 0ull;
    const double w = sample_weight(x, rs);
    return w >= minw || c == top ? sample_mass(w) : 0ull;
  };
  __syncthreads();
  sh.hist[2 * tid] = 0;
  sh.hist[2 * tid + 1] = 0;
  __syncthreads();
  row.each_chunk([&](int c, float (&y)[4], int i0) {
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < a.V) s += mass(y[j], i0 + j);
    s = wave_sum_u64(s);
    if (lane == 0) sh.hist[c * NW + wave] = s;
  });
  __syncthreads();
  // the segment of the token: the first whose end exceeds u x the whole (u >= 1: the last with any mass)
  const u64 ha = sh.hist[2 * tid], hb = sh.hist[2 * tid + 1];
  const u64 inw = wave_before_u64(ha + hb, lane);
  if (lane == 63) sh.red[wave] = inw + ha + hb;
  __syncthreads();
  u64 off = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    off += w < wave ? sh.red[w] : 0;
    all += sh.red[w];
  }
  const double want = (double)u * (double)all;
  const u64 lo = off + inw;
  auto inside = [&](u64 from, u64 m) -> bool {
    return m > 0 && (!((double)from > want) || from == 0) && ((double)(from + m) > want || from + m == all);
  };
  if (inside(lo, ha)) { sh.bin = 2 * tid; sh.before = lo; }
  if (inside(lo + ha, hb)) { sh.bin = 2 * tid + 1; sh.before = lo + ha; }
  __syncthreads();
  const int seg = sh.bin;
  if (wave != seg % NW) return;
  row.each_chunk([&](int c, float (&y)[4], int i0) {
    if (c != seg / NW) return;
    u64 m[4], s = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = i0 + j < a.V ? mass(y[j], i0 + j) : 0ull;
      s += m[j];
    }
    u64 at = sh.before + wave_before_u64(s, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (inside(at, m[j])) a.out[b] = i0 + j;
      at += m[j];
    }
  });
}

template <typename T>
int launch_sample(const SampleArgs& a, long long rows, hipStream_t st) {
  const dim3 grid((unsigned)rows);
  const int chunks = (a.V + 4 * ST - 1) / (4 * ST);
  if (chunks <= ROW_CHUNKS) {
    const size_t bytes = (size_t)chunks * 16 * ST;
    if (bytes > 32 * 1024) {
      const hipError_t e = hipFuncSetAttribute((const void*)sample_rows_kernel<T, true>,
                                               hipFuncAttributeMaxDynamicSharedMemorySize, ROW_CHUNKS * 16 * ST);
      if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL((sample_rows_kernel<T, true>), grid, dim3(ST), bytes, st, a);
  } else {
    hipLaunchKernelGGL((sample_rows_kernel<T, false>), grid, dim3(ST), 0, st, a);
  }
  NSP_LAUNCH_CHECK();
  return NSP_OK;
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
  if (s->dtype == NSP_DT_F32) return launch_sample<float>(a, s->rows, (hipStream_t)stream);
  if (s->dtype == NSP_DT_BF16) return launch_sample<__bf16>(a, s->rows, (hipStream_t)stream);
  return NSP_EUNSUPPORTED;
}
