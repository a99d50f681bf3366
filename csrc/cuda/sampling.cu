// Drawing one item per row from its scores (sm_100a): temperature, top-k, top-p, min-p, one given uniform number per row.
//
//   w_i = exp((x_i - max) / T);  in the order (score descending, index ascending) keep
//     the first k;  of those, up to the first whose running sum reaches p times their sum;  of those, w_i >= min_p
//   -> the smallest index i whose running sum over the kept items, in index order, exceeds u times their sum.
//
// Every filter keeps a beginning of the same order, so no sort is needed: histograms find the last kept value (by count for k,
// by weight for p) and how many of the items that share it are kept.
//   16-bit scores: the histogram has a bin for each of the 65536 patterns, 16-bit counts (a row where one passes 65535 is noticed
//     by their sum and done the other way).  The weights of the patterns that occur, some hundreds, are all that is computed;
//     afterwards they take the counts' place as a table, and the draw reads them from there.
//   fp32: bins of 1/64 octave of the weight, and a radix descent inside the bin that the cut falls into.
// Where at most LIST items can be kept (short rows, small k), one CTA sorts those instead.
//
// Weights are computed and summed in 64 bits: with N kept items each of the N borders can go either way with the sums'
// relative error as its chance, and 32-bit exponentials (1e-7 each) would draw a neighbour in every hundredth row of 10^5
// items.  The exponential is table-driven (Tang, ACM TOMS 15, 1989): 2^(n/256) from a table, 2^(f/256), |f| <= 1/2, as a
// polynomial of degree 3 (relative error (ln2/512)^4 / 24 = 1.4e-13).  Sums inside the histograms are whole numbers, so atomics in
// any order give the same bits: units of 2^-44 of the largest weight for rows up to 2^18 items, of about 2^-61 of the row's sum of weights
// beyond, which takes a rough look at that sum first.
//
// A row is read from memory once, into the shared memory of a cluster of CTAs (1 to 8 by its size and by how many rows there
// are), which then exchange histograms and sums through distributed shared memory; rows that do not fit are read again from
// L2.  Bound: for many long rows shared memory (one CTA, 131071 bf16 items, 73000 cycles: counting 19000, the draw's sums out of
// the table 26500, everything else 27500) and the waits of 16 warps for it, not the memory; in fp32 the histogram's atomics and the 64-bit arithmetic, ten
// operations per item and pass; for few or short rows the chain of short steps between the passes.
#include <cooperative_groups.h>

#include "common.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int NT = 512, NWARP = NT / 32;
constexpr int BINS = 2048, PB = BINS / NT;
constexpr int MAX_CLUSTER = 8;
constexpr int TABLE = 256;
constexpr int LIST = 1024;                      // items that are sorted, or kept aside for a descent
constexpr int GROUP = 64, GROUPS = 65536 / GROUP;   // 16-bit patterns are looked through in groups
constexpr int COUNT_BYTES = 65536 * 2;
constexpr int SLOTS = COUNT_BYTES / 8 / GROUP;  // groups whose weights fit where the counts were; the first holds zeros

struct SampleArgs {
  const void* scores; long long ld;             // dense: rows of `width`, `ld` elements apart
  const void* offsets; int offsets64;           // jagged: [rows + 1] into scores (then `width` is its length), or null
  long long width; int rows;
  int cap;                                      // elements of a slice that shared memory holds
  int counted;                                  // count the patterns (16-bit scores, one CTA per row)
  const float* uniform;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p;   // per row, or null: the values below
  float temperature_v; int top_k_v; float top_p_v, min_p_v;
  long long* ids; float* logprobs;
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// bits whose unsigned order is the order of the scores; NaN counts as -inf, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0x007fffffu;                                  // key of -inf
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t KEY_NONE = 0x007fffffu;                         // -inf: never drawn

// The same for the patterns of a 16-bit type, two at a time; NaN are the patterns outside (-inf, inf], -0 is next to 0.
__device__ __forceinline__ uint32_t patterns_of(uint32_t two) { return two ^ (((two >> 15) & 0x00010001u) * 0xffffu | 0x80008000u); }
template <typename T> __device__ __forceinline__ float pattern_value(uint32_t k) {
  const unsigned short b = static_cast<unsigned short>(k ^ ((k >> 15) ? 0x8000u : 0xffffu));
  return to_f<T>(*reinterpret_cast<const T*>(&b));
}
template <typename T> constexpr uint32_t INF16 = 0;                // the pattern of inf; its group holds no other number
template <> constexpr uint32_t INF16<__nv_bfloat16> = 0xff80u;
template <> constexpr uint32_t INF16<__half> = 0xfc00u;
constexpr uint32_t ZERO16 = 0x8000u;

// What the CTAs of a cluster read of one another
struct __align__(16) Shared {
  unsigned int lo[BINS], hi[BINS];              // 64-bit sums (or counts, in lo) by bin
  double table[TABLE];                          // 2^(j / TABLE)
  unsigned int best, first;                     // largest key of the slice; its first index (where that is all that is asked)
  unsigned long long list[LIST];                // (index, key) of the items that can be kept, or keys in the cut's bin
  unsigned int listed;
  unsigned int key_min, key_max;                // of the slice's items in the cut's bin
  double sum; unsigned int ties;                // of the slice's kept items; of those that equal the cut
  // within the CTA
  double wsum[NWARP];
  unsigned int wcnt[NWARP];
  unsigned long long wmass[NWARP];
  float queue[NWARP][64];
  unsigned int u0, u1, u2;
  unsigned long long m0, m1;
};

// exp((x - top) / T), 64 bits
struct Weigher {
  const double* table;
  double rate;                                  // 1 / T
  float top;
  // with its binary exponent raised by `up`; x is not NaN and at most top
  __device__ __forceinline__ double operator()(float x, int up = 0) const {
    const double t = x == top ? 0.0 : (static_cast<double>(x) - static_cast<double>(top)) * rate;
    const double magic = 6755399441055744.0;                       // 1.5 * 2^52: the sum's low word is the nearest whole number
    const double nd = fma(t, TABLE * 1.4426950408889634, magic);
    const int n = __double2loint(nd);
    const double f = fma(nd - magic, -0.6931471805599453 / TABLE, t);              // (next to 0 it is t itself: 1 - t is rounded once)
    const double q = fma(fma(fma(1.0 / 6.0, f, 0.5), f, 1.0), f, 1.0) * table[n & (TABLE - 1)];
    const double w = __hiloint2double(__double2hiint(q) + (((n >> 8) + up) << 20), __double2loint(q));
    return t > -700.0 ? w : 0.0;                                   // (2^-1010; also for -inf)
  }
  // the weight in units of 2^-up, rounded (up <= 61; the passes over all items know whether it is `small`, up to 51)
  __device__ __forceinline__ unsigned long long fixed(float x, int up) const {
    return up > 51 ? __double2ull_rn((*this)(x, up)) : small_fixed(x, up);
  }
  __device__ __forceinline__ unsigned long long small_fixed(float x, int up) const {
    const double w = (*this)(x, up) + 4503599627370496.0;          // + 2^52
    return static_cast<unsigned long long>(__double_as_longlong(w)) & 0xfffffffffffffULL;
  }
};

// In which units a row's weights are summed: 64 bits hold the sum.  Rows of up to SHORT items fit whatever their weights are; the
// sum of a longer one may be far below its number of items, and many weights that are nothing in units made for the latter can
// matter together.
constexpr int SHORT = 1 << 18, SHORT_SHIFT = 62 - 18;
__device__ __forceinline__ float rough_weight(float x, float top, float temp) {
  const float t = (x - top) * (1.44269504f / temp);
  return x == top ? 1.f : t > -150.f ? exp2f(t) : 0.f;            // (0 where t is NaN)
}
__device__ __forceinline__ int shift_for(double rough_sum) {      // (an upper bound of it, as a power of two)
  return 62 - max(1, (__double2hiint(rough_sum * 1.01) >> 20) - 1022);
}

// Where the order is cut: everything above `key` is kept and the first `ties` items (in index order) that equal it.
struct Cut { uint32_t key; unsigned int ties; };

__device__ __forceinline__ void add64(Shared& s, int bin, unsigned long long v) {
  const unsigned int lo = static_cast<unsigned int>(v);
  const unsigned int old = atomicAdd(&s.lo[bin], lo);
  const unsigned int hi = static_cast<unsigned int>(v >> 32) + (old + lo < old ? 1u : 0u);
  if (hi) atomicAdd(&s.hi[bin], hi);
}

// f(scores, how many, index of the first in the slice) for all of a slice, 16 bytes at a time where its address allows
template <typename T, typename F>
__device__ __forceinline__ void for_each(const T* x, int n, F&& f) {
  constexpr int V = 16 / sizeof(T);
  const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)));
  const int nv = (n - head) / V;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  for (int i = threadIdx.x; i < nv; i += NT) {
    const uint4 u = xv[i];
    const T* e = reinterpret_cast<const T*>(&u);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f<T>(e[j]);
    f(v, head + i * V);
  }
  // the ends, one by one
  const int ends = n - nv * V;
  if (static_cast<int>(threadIdx.x) < ends) {
    const int i = static_cast<int>(threadIdx.x) < head ? threadIdx.x : nv * V + threadIdx.x;
    float v[1] = {to_f<T>(x[i])};
    f(v, i);
  }
}

template <typename T>
__global__ void __launch_bounds__(NT, 1) sample_kernel(const SampleArgs p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  unsigned int* counts = reinterpret_cast<unsigned int*>(smem + (sizeof(Shared) + 15) / 16 * 16);   // two to a word
  T* store = reinterpret_cast<T*>(smem + (sizeof(Shared) + 15) / 16 * 16 + (p.counted ? COUNT_BYTES : 0));
  cg::cluster_group cluster = cg::this_cluster();
  const int c = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < TABLE; i += NT) s.table[i] = exp2(i / static_cast<double>(TABLE));
  auto sync = [&]() { if (c > 1) cluster.sync(); else __syncthreads(); };
  auto peer = [&](int r) -> Shared& { return c > 1 ? *cluster.map_shared_rank(&s, r) : s; };

  for (int row = blockIdx.x / c; row < p.rows; row += gridDim.x / c) {
    long long lo = 0, hi = p.width;
    const T* x = reinterpret_cast<const T*>(p.scores);
    if (p.offsets) {
      lo = p.offsets64 ? static_cast<const long long*>(p.offsets)[row] : static_cast<const int*>(p.offsets)[row];
      hi = p.offsets64 ? static_cast<const long long*>(p.offsets)[row + 1] : static_cast<const int*>(p.offsets)[row + 1];
      lo = min(max(lo, 0LL), p.width);
      hi = min(max(hi, lo), p.width);
      x += lo;
    } else {
      x += row * p.ld;
    }
    const int n_row = static_cast<int>(hi - lo);
    // this CTA's slice [s_lo, s_lo + n)
    const int part = ((n_row + c - 1) / c + 31) / 32 * 32;
    const int s_lo = min(rank * part, n_row), n = min(part, n_row - s_lo);
    x += s_lo;
    const float temp = p.temperature ? p.temperature[row] : p.temperature_v;
    const int top_k = p.top_k ? p.top_k[row] : p.top_k_v;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_v;
    const float min_pv = p.min_p ? p.min_p[row] : p.min_p_v;
    const float min_p = min_pv == min_pv ? min_pv : 1.f;           // NaN: no weight is known to be enough but the largest
    const float uf = p.uniform[row];
    const double u = uf > 0.f ? static_cast<double>(uf) : 0.0;

    // ---- bring the slice in, with a look at each 16 bytes (`vec`) and at the ends (`one`)
    auto bring = [&](auto&& vec, auto&& one) {
      constexpr int V = 16 / sizeof(T);
      const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / static_cast<int>(sizeof(T)));
      const int nv = (n - head) / V;
      const bool keep = n <= p.cap;
      // at the same offset from a 16-byte border, so that both sides move in vectors
      T* y = store + (reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T);
      const uint4* xv = reinterpret_cast<const uint4*>(x + head);
      uint4* yv = reinterpret_cast<uint4*>(y + head);
#pragma unroll 4
      for (int i = tid; i < nv; i += NT) {
        const uint4 v = __ldg(xv + i);
        if (keep) yv[i] = v;
        vec(v);
      }
      const int ends = n - nv * V;
      if (tid < ends) {
        const int i = tid < head ? tid : nv * V + tid;
        if (keep) y[i] = x[i];
        one(x[i]);
      }
      if (keep) x = y;
    };

    int shift_fx = SHORT_SHIFT;
    // of the CTA, the same bits for all
    auto sum_of_all = [&](double v) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      __syncthreads();
      if (lane == 0) s.wsum[warp] = v;
      __syncthreads();
      v = 0.0;
      for (int i = 0; i < NWARP; ++i) v += s.wsum[i];
      __syncthreads();
      return v;
    };

    // ---- 16-bit scores: how often each pattern occurs is all that the cuts need
    uint32_t top_key = 0, top16 = 0, cut16 = 0;
    Cut cut = {KEY_NONE, 0};
    bool counted = false;
    unsigned short* slot = reinterpret_cast<unsigned short*>(s.lo + GROUPS);       // by group: where its weights are
    unsigned short* group = slot + GROUPS;                         // those that are not empty, from the highest down
    int groups = 0;
    if constexpr (sizeof(T) == 2) {
      if (p.counted && temp > 0.f && n_row > LIST && !(top_k > 0 && top_k <= LIST / 2)) {
        unsigned int* in_group = s.lo;
        unsigned long long* mass = reinterpret_cast<unsigned long long*>(s.hi);    // of a group
        for (int i = tid; i < COUNT_BYTES / 16; i += NT) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        auto count = [&](uint32_t k) { atomicAdd(counts + (k >> 1), (k & 1) ? 0x10000u : 1u); };
        auto count2 = [&](uint32_t two) {
          const uint32_t k = patterns_of(two);
          count(k & 0xffffu);
          count(k >> 16);
        };
        bring([&](const uint4& v) { count2(v.x); count2(v.y); count2(v.z); count2(v.w); },
              [&](const T& v) { count(patterns_of(*reinterpret_cast<const unsigned short*>(&v)) & 0xffffu); });
        __syncthreads();
        if (tid == 0) {
          s.u0 = 0; s.u1 = 0;
          // -0 is 0
          const unsigned int minus = counts[ZERO16 / 2 - 1] >> 16;
          if (minus + (counts[ZERO16 / 2] & 0xffffu) > 0xffffu) {
            s.u1 = 1;
          } else {
            counts[ZERO16 / 2 - 1] &= 0xffffu;
            counts[ZERO16 / 2] += minus;
          }
        }
        __syncthreads();
        constexpr int g_inf = INF16<T> / GROUP, g_none = (0xffffu - INF16<T>) / GROUP;
        unsigned int seen = 0;
        int g_top = 0;
#pragma unroll 4
        for (int i = tid; i < COUNT_BYTES / 16; i += NT) {         // 8 threads per group
          uint4 w = reinterpret_cast<const uint4*>(counts)[i];
          const int g = i / (GROUP / 8);
          seen += (w.x & 0xffffu) + (w.x >> 16) + (w.y & 0xffffu) + (w.y >> 16) + (w.z & 0xffffu) + (w.z >> 16) + (w.w & 0xffffu) + (w.w >> 16);
          if (g >= g_inf || g <= g_none) {
            w = make_uint4(g == g_inf && i % (GROUP / 8) == 0 ? w.x & 0xffffu : 0, 0, 0, 0);
            reinterpret_cast<uint4*>(counts)[i] = w;
          }
          unsigned int m = (w.x & 0xffffu) + (w.x >> 16) + (w.y & 0xffffu) + (w.y >> 16) + (w.z & 0xffffu) + (w.z >> 16) + (w.w & 0xffffu) + (w.w >> 16);
          m += __shfl_xor_sync(0xffffffffu, m, 1);
          m += __shfl_xor_sync(0xffffffffu, m, 2);
          m += __shfl_xor_sync(0xffffffffu, m, 4);
          if (i % (GROUP / 8) == 0) in_group[g] = m;
          if (m) g_top = max(g_top, g);
        }
        seen = __reduce_add_sync(0xffffffffu, seen);
        g_top = __reduce_max_sync(0xffffffffu, g_top);
        if (lane == 0) { s.wcnt[warp] = seen; atomicMax(&s.u0, g_top); }
        __syncthreads();
        seen = 0;
        for (int i = 0; i < NWARP; ++i) seen += s.wcnt[i];
        // A count that passed 16 bits took 65535 or 65536 from the sum: such a row is done by weight, below.
        counted = seen == static_cast<unsigned int>(n_row) && !s.u1;
        g_top = s.u0;
        __syncthreads();
        if (counted) {
          const unsigned int wt_ = counts[g_top * 32 + lane];
          top16 = g_top * GROUP + __reduce_max_sync(0xffffffffu, (wt_ >> 16) ? 2 * lane + 1 : wt_ ? 2 * lane : 0);
          if (in_group[g_top] == 0) {
            if (tid == 0) { p.ids[row] = -1; p.logprobs[row] = -INFINITY; }
            __syncthreads();
            continue;
          }
          const float top_f = pattern_value<T>(top16);
          top_key = key_of(top_f);
          Weigher wt;
          wt.table = s.table; wt.top = top_f;
          wt.rate = 1.0 / static_cast<double>(temp);
          // list the groups, two per thread (and always -0's, for its weight)
          static_assert(GROUPS == 2 * NT, "two groups per thread");
          {
            const int g = GROUPS - 1 - 2 * tid;
            const bool f0 = in_group[g] || g == ZERO16 / GROUP - 1, f1 = in_group[g - 1] != 0;
            const unsigned int b0 = __ballot_sync(0xffffffffu, f0), b1 = __ballot_sync(0xffffffffu, f1);
            if (lane == 0) s.wcnt[warp] = __popc(b0) + __popc(b1);
            __syncthreads();
            int at = __popc(b0 & ((1u << lane) - 1)) + __popc(b1 & ((1u << lane) - 1));
            for (int i = 0; i < NWARP; ++i) {
              if (i < warp) at += s.wcnt[i];
              groups += s.wcnt[i];
            }
            if (f0) group[at++] = g;
            if (f1) group[at] = g - 1;
            __syncthreads();
          }
          for (int by_mass = 0; by_mass < 2; ++by_mass) {
            if (by_mass ? !(top_p < 1.f) : !(top_k > 0 && top_k < n_row)) continue;
            if (by_mass && n_row > SHORT) {
              double rough = 0.0;
              for (int i = tid; i < groups * (GROUP / 2); i += NT) {
                const int at = group[i / (GROUP / 2)] * (GROUP / 2) + i % (GROUP / 2);
                const unsigned int w = counts[at];
                if (w & 0xffffu) rough += static_cast<double>(w & 0xffffu) * rough_weight(pattern_value<T>(2 * at), top_f, temp);
                if (w >> 16) rough += static_cast<double>(w >> 16) * rough_weight(pattern_value<T>(2 * at + 1), top_f, temp);
              }
              shift_fx = shift_for(sum_of_all(rough));
            }
            auto kept = [&](uint32_t k, unsigned int m) -> unsigned int { return k > cut16 ? m : k == cut16 ? cut.ties : 0; };
            auto value = [&](uint32_t k, unsigned int m) -> unsigned long long {
              return kept(k, m) * (by_mass ? wt.fixed(pattern_value<T>(k), shift_fx) : 1ULL);
            };
            auto sum_groups = [&](auto units) {
              // eight threads per group, eight patterns each
              for (int i = tid; i < (groups * (GROUP / 8) + 31) / 32 * 32; i += NT) {
                const int at = i / (GROUP / 8);
                const int k = group[min(at, groups - 1)] * GROUP + i % (GROUP / 8) * 8;
                const uint4 w = *reinterpret_cast<const uint4*>(counts + k / 2);
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
                unsigned long long v = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) v += kept(k + j, j & 1 ? ws[j / 2] >> 16 : ws[j / 2] & 0xffffu) * units(k + j);
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                v += __shfl_xor_sync(0xffffffffu, v, 4);
                if (i % (GROUP / 8) == 0 && at < groups) mass[at] = v;
              }
            };
            if (!by_mass) sum_groups([](uint32_t) { return 1ULL; });
            else if (n_row <= SHORT) sum_groups([&](uint32_t k) { return wt.small_fixed(pattern_value<T>(k), SHORT_SHIFT); });
            else sum_groups([&](uint32_t k) { return wt.fixed(pattern_value<T>(k), shift_fx); });
            if (tid == 0) s.u2 = 0;
            __syncthreads();
            const unsigned long long v0 = 2 * tid < groups ? mass[2 * tid] : 0, v1 = 2 * tid + 1 < groups ? mass[2 * tid + 1] : 0;
            unsigned long long incl = v0 + v1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
              if (lane >= o) incl += y;
            }
            if (lane == 31) s.wmass[warp] = incl;
            __syncthreads();
            unsigned long long before = incl - v0 - v1, all = 0, target;
            for (int i = 0; i < NWARP; ++i) {
              if (i < warp) before += s.wmass[i];
              all += s.wmass[i];
            }
            if (by_mass) {
              const double t = ceil(static_cast<double>(top_p) * static_cast<double>(all));
              target = t > 1.0 ? static_cast<unsigned long long>(t) : 1ULL;        // at least the first item
            } else {
              target = all <= static_cast<unsigned int>(top_k) ? ~0ULL : static_cast<unsigned long long>(top_k);
            }
            if (before < target && before + v0 >= target) { s.u0 = group[2 * tid]; s.m0 = before; s.u2 = 1; }
            before += v0;
            if (before < target && before + v1 >= target) { s.u0 = group[2 * tid + 1]; s.m0 = before; s.u2 = 1; }
            __syncthreads();
            if (s.u2) {
              // its patterns, two per lane from the highest down
              const int at = s.u0 * 32 + 31 - lane;
              const unsigned int w = counts[at], k = 2 * at;
              const unsigned long long a1 = value(k + 1, w >> 16), a0 = value(k, w & 0xffffu);
              unsigned long long run = a0 + a1;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long y = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += y;
              }
              unsigned long long above = s.m0 + run - a0 - a1;
              const int who = __ffs(__ballot_sync(0xffffffffu, s.m0 + run >= target)) - 1;
              const bool second = above + a1 < target;
              if (second) above += a1;
              const unsigned int key = k + (second ? 0 : 1);
              unsigned long long kept = target - above;
              if (by_mass) {
                const unsigned long long one = wt.fixed(pattern_value<T>(key), shift_fx);
                const unsigned int most = key == cut16 ? cut.ties : 0xffffffffu;
                kept = one ? min((kept + one - 1) / one, static_cast<unsigned long long>(most)) : most;
              }
              cut.ties = __shfl_sync(0xffffffffu, static_cast<unsigned int>(kept), who);
              cut16 = __shfl_sync(0xffffffffu, key, who);
              cut.key = key_of(pattern_value<T>(cut16));
            }
            __syncthreads();
          }
        }
      }
    }
    if (!counted) {
      float most = -INFINITY;                                      // (fmaxf passes over NaN)
      bring([&](const uint4& v) {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < static_cast<int>(16 / sizeof(T)); ++j) most = fmaxf(most, to_f<T>(e[j]));
      }, [&](const T& v) { most = fmaxf(most, to_f<T>(v)); });
      top_key = __reduce_max_sync(0xffffffffu, key_of(most));
      if (lane == 0) s.wcnt[warp] = top_key;
    }
    if (tid == 0) { s.listed = 0; s.first = 0xffffffffu; }
    __syncthreads();
    if (tid == 0) {
      if (!counted) for (int i = 0; i < NWARP; ++i) top_key = max(top_key, s.wcnt[i]);
      s.best = top_key;
    }
    sync();
    for (int r = 0; r < c; ++r) top_key = max(top_key, peer(r).best);
    if (n_row == 0 || top_key <= KEY_NONE) {
      if (rank == 0 && tid == 0) { p.ids[row] = -1; p.logprobs[row] = -INFINITY; }
      sync();                                                      // nobody's words are still being read
      continue;
    }
    if (!(temp > 0.f)) {
      unsigned int at = 0xffffffffu;
      const float top_f = value_of(top_key);
      for_each<T>(x, n, [&](auto& v, int i) {
        for (float e : v) {
          if (e == top_f) at = min(at, static_cast<unsigned int>(s_lo + i));
          ++i;
        }
      });
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0 && at != 0xffffffffu) atomicMin(&peer(0).first, at);
      sync();
      if (rank == 0 && tid == 0) { p.ids[row] = s.first; p.logprobs[row] = 0.f; }
      sync();
      continue;
    }
    const float top_f = value_of(top_key);
    Weigher wt;
    wt.table = s.table; wt.top = top_f;
    wt.rate = 1.0 / static_cast<double>(temp);
    auto wk = [&](uint32_t k) { return wt(value_of(k)); };
    float cut_f = value_of(cut.key);
    // bins of 1/64 octave of the weight, the last one open: all that matters is that they are monotone in the score
    const float bin_scale = 64.f * 1.44269504f / temp, bin_shift = top_f * bin_scale;
    auto place_of = [&](float x) { return fmaxf(fminf(fmaf(x, -bin_scale, bin_shift), BINS - 1.f), 0.f); };
    auto bin_of = [&](float x) { return static_cast<int>(place_of(x)); };
    const double mp = static_cast<double>(min_p);
    auto enough = [&](double w) { return w >= mp && mp < 1.0; };   // next to the largest score the weight rounds to 1, but is less

    // ---- the first CTA's list holds everything that can be kept, `m` items (index, key): sorted keys give the cut, the
    // draw goes through the items in index order, in which the list is already or is brought first.
    auto draw_listed = [&](int m, bool ordered) {
      int size = 2;
      while (size < m) size *= 2;
      const int i0 = 2 * tid, i1 = i0 + 1;
      const bool busy = warp * 64 < size;                          // has items
      // bitonic by index, two neighbouring items per thread: partners up to 32 apart are in the warp, others are met in the list
      auto sort_list = [&](unsigned long long& v0, unsigned long long& v1) {
        for (int k = 2; k <= size; k *= 2) {
          const bool up = (i0 & k) == 0;                           // the smaller of a pair comes first
          for (int j = k / 2; j >= 64; j /= 2) {
            __syncthreads();
            if (i0 < size) { s.list[i0] = v0; s.list[i1] = v1; }
            __syncthreads();
            if (i0 < size) {
              const unsigned long long q0 = s.list[i0 ^ j], q1 = s.list[i1 ^ j];
              const bool smaller = ((i0 & j) == 0) == up;
              v0 = smaller ? min(v0, q0) : max(v0, q0);
              v1 = smaller ? min(v1, q1) : max(v1, q1);
            }
          }
          if (!busy) continue;
          for (int j = min(k / 2, 32); j > 1; j /= 2) {
            const unsigned long long q0 = __shfl_xor_sync(0xffffffffu, v0, j / 2), q1 = __shfl_xor_sync(0xffffffffu, v1, j / 2);
            const bool smaller = ((i0 & j) == 0) == up;
            v0 = smaller ? min(v0, q0) : max(v0, q0);
            v1 = smaller ? min(v1, q1) : max(v1, q1);
          }
          const unsigned long long lo = min(v0, v1), hi = max(v0, v1);
          v0 = up ? lo : hi;
          v1 = up ? hi : lo;
        }
      };
      // bitonic, from the largest down, eight neighbouring keys per thread of the first four warps (one for each of the SM's
      // four schedulers): most partners are in the thread or the warp.  1024 keys: 6200 cycles, with two per thread 7600.
      auto sort_keys = [&](uint32_t* keys) {
        if (warp < 4) {
          const int n = max(size, 8), at = 8 * tid;
          const bool mine = at < n;
          uint32_t v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = mine ? keys[at + e] : 0u;
          auto within = [&](int j, auto down) {                    // partners of one thread
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (e & j) continue;
              const uint32_t hi = max(v[e], v[e | j]), lo = min(v[e], v[e | j]);
              v[e] = down(e) ? hi : lo;
              v[e | j] = down(e) ? lo : hi;
            }
          };
          within(1, [](int e) { return (e & 2) == 0; });
          within(2, [](int e) { return (e & 4) == 0; });
          within(1, [](int e) { return (e & 4) == 0; });
          for (int k = 8; k <= n; k *= 2) {
            const bool down = (at & k) == 0;
            for (int j = k / 2; j >= 256; j /= 2) {
              rb::named_barrier(1, 128);
              if (mine) {
#pragma unroll
                for (int e = 0; e < 8; ++e) keys[at + e] = v[e];
              }
              rb::named_barrier(1, 128);
              if (mine) {
                const bool larger = ((at & j) == 0) == down;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const uint32_t q = keys[(at ^ j) + e];
                  v[e] = larger ? max(v[e], q) : min(v[e], q);
                }
              }
            }
            for (int j = min(k / 2, 128); j >= 8; j /= 2) {
              const bool larger = ((at & j) == 0) == down;
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t q = __shfl_xor_sync(0xffffffffu, v[e], j / 8);
                v[e] = larger ? max(v[e], q) : min(v[e], q);
              }
            }
            auto one_way = [&](int) { return down; };
            within(4, one_way);
            within(2, one_way);
            within(1, one_way);
          }
          rb::named_barrier(1, 128);
          if (mine) {
#pragma unroll
            for (int e = 0; e < 8; ++e) keys[at + e] = v[e];
          }
        }
        __syncthreads();
      };
      // running sums of two items per thread, in order -> sum before the first of them
      auto scan = [&](double w0, double w1, double& all) {
        double incl = w0 + w1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        __syncthreads();
        if (lane == 31) s.wsum[warp] = incl;
        __syncthreads();
        double before = __shfl_up_sync(0xffffffffu, incl, 1);
        if (lane == 0) before = 0.0;
        double sums = lane < NWARP ? s.wsum[lane] : 0.0;
#pragma unroll
        for (int o = 1; o < NWARP; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, sums, o);
          if (lane >= o) sums += y;
        }
        all = __shfl_sync(0xffffffffu, sums, NWARP - 1);
        const double earlier = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0));
        return warp ? before + earlier : before;
      };
      unsigned long long e0 = i0 < m ? s.list[i0] : ~0ULL << 32, e1 = i1 < m ? s.list[i1] : ~0ULL << 32;
      if (!ordered) sort_list(e0, e1);
      const uint32_t key0 = static_cast<uint32_t>(e0), key1 = static_cast<uint32_t>(e1);
      uint32_t* keys = s.hi;
      keys[i0] = key0;
      keys[i1] = key1;
      __syncthreads();
      sort_keys(keys);
      const uint32_t k0 = keys[i0], k1 = keys[i1];
      auto item = [&](int i, uint32_t k) { return k > KEY_NONE && (top_k <= 0 || i < top_k) ? wk(k) : 0.0; };
      const double w0 = item(i0, k0), w1 = item(i1, k1);
      double all, kept_all;
      const double before = scan(w0, w1, all);
      const double limit = top_p < 1.f ? static_cast<double>(top_p) * all : INFINITY;
      auto kept = [&](int i, uint32_t k, double w, double b) {
        return k > KEY_NONE && (top_k <= 0 || i < top_k) && (i == 0 || b < limit) && (enough(w) || k == top_key);
      };
      const int n_kept = __syncthreads_count(kept(i0, k0, w0, before)) + __syncthreads_count(kept(i1, k1, w1, before + w0));
      const uint32_t last = keys[n_kept - 1];                      // (the largest score is always kept)
      const int ties = n_kept - __syncthreads_count(k0 > last) - __syncthreads_count(k1 > last);
      // in index order
      const unsigned int b0 = __ballot_sync(0xffffffffu, key0 == last), b1 = __ballot_sync(0xffffffffu, key1 == last);
      if (lane == 0) s.wcnt[warp] = __popc(b0) + __popc(b1);
      __syncthreads();
      int tied = __popc(b0 & ((1u << lane) - 1)) + __popc(b1 & ((1u << lane) - 1));
      for (int i = 0; i < warp; ++i) tied += s.wcnt[i];
      const double v0 = key0 > last || (key0 == last && tied < ties) ? wk(key0) : 0.0;
      const double v1 = key1 > last || (key1 == last && tied + (key0 == last) < ties) ? wk(key1) : 0.0;
      const double run = scan(v0, v1, kept_all);
      const double target = u * kept_all;
      if (tid == 0) { s.u0 = 0xffffffffu; s.u1 = 0; }
      __syncthreads();
      if (v0 > 0.0) { if (run + v0 > target) atomicMin(&s.u0, i0); atomicMax(&s.u1, i0); }
      if (v1 > 0.0) { if (run + v0 + v1 > target) atomicMin(&s.u0, i1); atomicMax(&s.u1, i1); }
      __syncthreads();
      const unsigned int pick = s.u0 != 0xffffffffu ? s.u0 : s.u1;
      if (i0 == (pick & ~1u)) {
        p.ids[row] = static_cast<long long>((pick & 1 ? e1 : e0) >> 32);
        p.logprobs[row] = static_cast<float>(log((pick & 1 ? v1 : v0) / kept_all));
      }
    };
    auto entry = [&](uint32_t k, int i) { return static_cast<unsigned long long>(s_lo + i) << 32 | k; };
    auto list_item = [&](uint32_t k, int i) {
      Shared& first = peer(0);
      const unsigned int at = atomicAdd(&first.listed, 1u);
      if (at < LIST) first.list[at] = entry(k, i);
    };
    if (n_row <= LIST) {
      unsigned long long* list = peer(0).list + s_lo;
      for_each<T>(x, n, [&](auto& v, int i) {
        for (float e : v) {
          list[i] = entry(key_of(e), i);
          ++i;
        }
      });
      sync();
      if (rank == 0) draw_listed(n_row, true);
      sync();
      continue;
    }
    bool drawn = false;

    for (int by_mass = 0; by_mass < 2 && !drawn && !counted; ++by_mass) {
      if (by_mass ? !(top_p < 1.f) : !(top_k > 0 && top_k < n_row)) continue;
      // Finds, from the top, the bin where the running sum reaches the target.  -> u2: found, u0: the bin, u1 / m0: what is above it
      unsigned long long target = 0, above = 0, in_bin = 0, all = 0;
      auto find_bin = [&](bool upwards) {
        // the cluster's histogram, PB bins per thread in order from the highest score down
        static_assert(PB == 4, "a thread's bins are one vector");
        unsigned long long v[PB] = {0, 0, 0, 0}, mine = 0;
        const int at = upwards ? tid : BINS / PB - 1 - tid;
        auto add4 = [&](const uint4& l, int shift) {
          const uint32_t ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] += static_cast<unsigned long long>(ls[i]) << shift;
        };
        for (int r = 0; r < c; r += 4) {                           // four peers' loads in flight; counts have no high words
          uint4 l[4], h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            l[i] = h[i] = make_uint4(0, 0, 0, 0);
            if (r + i < c) {
              const Shared& a = peer(r + i);
              l[i] = reinterpret_cast<const uint4*>(a.lo)[at];
              if (by_mass) h[i] = reinterpret_cast<const uint4*>(a.hi)[at];
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) { add4(l[i], 0); add4(h[i], 32); }
        }
        if (!upwards) {
          unsigned long long y = v[0]; v[0] = v[3]; v[3] = y;
          y = v[1]; v[1] = v[2]; v[2] = y;
        }
        mine = v[0] + v[1] + v[2] + v[3];
        unsigned long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        if (lane == 31) s.wmass[warp] = incl;
        if (tid == 0) s.u2 = 0;
        __syncthreads();
        unsigned long long before = above + incl - mine;
        all = 0;
        for (int i = 0; i < NWARP; ++i) {
          if (i < warp) before += s.wmass[i];
          all += s.wmass[i];
        }
        if (!target) {
          if (by_mass) {
            const double t = ceil(static_cast<double>(top_p) * static_cast<double>(all));
            target = t > 1.0 ? static_cast<unsigned long long>(t) : 1ULL;     // at least the first item
          } else {
            target = all <= static_cast<unsigned int>(top_k) ? ~0ULL : static_cast<unsigned long long>(top_k);
          }
        }
#pragma unroll
        for (int i = 0; i < PB; ++i) {
          if (before < target && before + v[i] >= target) { s.u0 = upwards ? tid * PB + i : BINS - 1 - (tid * PB + i); s.m0 = before; s.m1 = v[i]; s.u2 = 1; }
          before += v[i];
        }
        __syncthreads();
        if (s.u2) { above = s.m0; in_bin = s.m1; }
        return s.u2 ? static_cast<int>(s.u0) : -1;
      };
      auto clear = [&]() {
        for (int i = tid; i < BINS; i += NT) { s.lo[i] = 0; s.hi[i] = 0; }
        if (tid == 0) { s.key_min = 0xffffffffu; s.key_max = 0; }
        __syncthreads();
      };
      auto add = [&](int bin, float e) {
        if (by_mass) add64(s, bin, wt.fixed(e, shift_fx)); else atomicAdd(&s.lo[bin], 1u);
      };
      // items equal to an earlier cut count as many times as they are kept: one thread adds them
      const bool lump = by_mass && cut.ties && rank == 0 && tid == 0;
      if (by_mass && n_row > SHORT) {
        double rough = 0.0;
        for_each<T>(x, n, [&](auto& v, int) {
          for (float e : v) rough += rough_weight(e, top_f, temp);
        });
        rough = sum_of_all(rough);
        if (tid == 0) s.sum = rough;
        sync();
        rough = 0.0;
        for (int r = 0; r < c; ++r) rough += peer(r).sum;
        shift_fx = shift_for(rough);
      }
      sync();                                                      // earlier histograms have been read
      clear();
      if (by_mass) {
        auto weigh = [&](auto units) {
          for_each<T>(x, n, [&](auto& v, int) {
            constexpr int N = sizeof(v) / sizeof(float);
            unsigned long long w[N];                               // all the arithmetic before the first atomic
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = units(v[j]);
#pragma unroll
            for (int j = 0; j < N; ++j) if (v[j] > cut_f) add64(s, bin_of(v[j]), w[j]);
          });
        };
        if (n_row <= SHORT) weigh([&](float e) { return wt.small_fixed(e, SHORT_SHIFT); });
        else weigh([&](float e) { return wt.fixed(e, shift_fx); });
      } else {
        for_each<T>(x, n, [&](auto& v, int) {
          for (float e : v) if (e > cut_f) atomicAdd(&s.lo[bin_of(e)], 1u);
        });
      }
      if (lump) add64(s, bin_of(cut_f), cut.ties * wt.fixed(cut_f, shift_fx));
      sync();
      const int bin = find_bin(true);
      if (bin < 0) continue;                                       // fewer items than k
      if (!by_mass && above + in_bin <= LIST) {                    // all that can be kept fits the list
        for_each<T>(x, n, [&](auto& v, int i) {
          for (float e : v) {
            if (e > -INFINITY && bin_of(e) <= bin) list_item(key_of(e), i);
            ++i;
          }
        });
        sync();
        if (rank == 0) draw_listed(static_cast<int>(s.listed), false);
        drawn = true;
        break;
      }
      // the keys in that bin (set aside while they are few), then a descent over their range
      uint32_t k_min = 0xffffffffu, k_max = 0;
      uint32_t* aside = reinterpret_cast<uint32_t*>(s.list);
      if (tid == 0) s.listed = 0;
      __syncthreads();
      auto in_this = [&](float e) {
        const float at = place_of(e);
        return e > cut_f && at >= bin && (at < bin + 1.f || bin == BINS - 1);
      };
      for_each<T>(x, n, [&](auto& v, int) {
        for (float e : v)
          if (in_this(e)) {
            const uint32_t k = key_of(e);
            k_min = min(k_min, k);
            k_max = max(k_max, k);
            const unsigned int at = atomicAdd(&s.listed, 1u);
            if (at < 2 * LIST) aside[at] = k;
          }
      });
      if (lump && bin_of(cut_f) == bin) { k_min = min(k_min, cut.key); k_max = max(k_max, cut.key); }
      k_min = __reduce_min_sync(0xffffffffu, k_min);
      k_max = __reduce_max_sync(0xffffffffu, k_max);
      if (lane == 0 && k_min <= k_max) { atomicMin(&s.key_min, k_min); atomicMax(&s.key_max, k_max); }
      sync();
      const int n_aside = static_cast<int>(s.listed);
      for (int r = 0; r < c; ++r) { k_min = min(k_min, peer(r).key_min); k_max = max(k_max, peer(r).key_max); }
      while (k_min < k_max) {
        const int down = max(0, 32 - __clz(k_max - k_min) - 11);   // (k_max - k_min) >> down < 2^11
        sync();
        clear();
        if (n_aside <= 2 * LIST) {
          for (int i = tid; i < n_aside; i += NT) {
            const uint32_t k = aside[i];
            if (k >= k_min && k <= k_max) add((k - k_min) >> down, value_of(k));
          }
        } else {
          for_each<T>(x, n, [&](auto& v, int) {
            for (float e : v) {
              if (!in_this(e)) continue;
              const uint32_t k = key_of(e);
              if (k >= k_min && k <= k_max) add((k - k_min) >> down, e);
            }
          });
        }
        if (lump && cut.key >= k_min && cut.key <= k_max && bin_of(cut_f) == bin)
          add64(s, (cut.key - k_min) >> down, cut.ties * wt.fixed(cut_f, shift_fx));
        sync();
        const int b = find_bin(false);
        if (b < 0) break;                                          // (cannot be: the sum is reached in this range)
        k_min += static_cast<uint32_t>(b) << down;
        k_max = min(k_max, k_min + ((1u << down) - 1u));
      }
      if (by_mass) {
        const unsigned long long w = wt.fixed(value_of(k_min), shift_fx);
        const unsigned long long r = w ? (target - above + w - 1) / w : 0xffffffffULL;
        const unsigned int most = k_min == cut.key ? cut.ties : 0xffffffffu;
        cut.ties = static_cast<unsigned int>(min(r, static_cast<unsigned long long>(most)));
      } else {
        cut.ties = static_cast<unsigned int>(target - above);
      }
      cut.key = k_min;
      cut_f = value_of(k_min);
    }

    if (drawn) {
      sync();
      continue;
    }
    // ---- draw: which CTA, which warp, ... holds the item where the running sum passes u * total
    // where patterns were counted, the kept ones' weights take the counts' place, if their groups fit
    bool tabled = false;
    double* weights = reinterpret_cast<double*>(counts);
    uint32_t tie16 = 0x10000u, tie16b = 0x10000u, low16 = 0;       // (0x10000: no pattern)
    if constexpr (sizeof(T) == 2) {
      if (counted) {
        auto in = [&](int i) { return i < groups && group[i] >= cut16 / GROUP; };      // the first of the list
        reinterpret_cast<uint32_t*>(slot)[tid] = 0;
        if (tid == 0) s.u2 = 0xffffu;
        const int used = 1 + __syncthreads_count(in(tid)) + __syncthreads_count(in(tid + NT));
        tabled = used <= SLOTS;
        if (tabled) {
          if (tid + 1 < used) slot[group[tid]] = tid + 1;
          uint32_t low = 0xffffu;
          for (int i = tid; i < used * GROUP; i += NT) {
            double w = 0.0;
            if (i >= GROUP) {
              const uint32_t k = group[i / GROUP - 1] * GROUP + i % GROUP;
              if (k > cut16 && k <= top16) {
                w = wt(pattern_value<T>(k));
                if (enough(w) || pattern_value<T>(k) == top_f) low = min(low, k); else w = 0.0;
              }
            }
            weights[i] = w;
          }
          low = __reduce_min_sync(0xffffffffu, low);
          if (lane == 0) atomicMin(&s.u2, low);
          __syncthreads();
          low16 = s.u2;
          if (cut.ties) {
            tie16 = cut16;
            tie16b = cut16 == ZERO16 ? ZERO16 - 1 : cut16;
          }
        }
      }
    }
    auto weight16 = [&](uint32_t k) { return weights[slot[k / GROUP] * GROUP + k % GROUP]; };
    // min-p as a key: the smallest one with enough weight, by 32 tries at a time
    uint32_t lim = cut.key;                                        // kept: keys above it, and the cut's ties
    if (mp > 0.0 && !tabled) {
      uint32_t below = mp < 1.0 ? KEY_NONE : top_key - 1, most = top_key;            // w(below) < mp <= w(most)
      if (mp < 1.0 && !isinf(top_f)) {
        // where it should be, give or take: a bracket that is checked before it is used
        const float guess = top_f + temp * __logf(min_p), slack = 1e-3f * (fabsf(temp) + 1e-3f * fabsf(guess));
        const float g0 = guess - slack, g1 = fminf(guess + slack, top_f);
        if (g0 > -INFINITY && g0 < g1 && wt(g0) < mp && wt(g1) >= mp) { below = key_of(g0); most = key_of(g1); }
      }
      while (most - below > 1) {
        const uint32_t step = (most - below - 1) / 32 + 1, k = below + step * (lane + 1);
        const unsigned int yes = __ballot_sync(0xffffffffu, k < most && k > below && wk(k) >= mp);
        const uint32_t tried = (most - below - 1) / step;        // tries below `most`; from the f-th on they have enough weight
        const uint32_t f = yes ? __ffs(yes) - 1 : tried;
        if (yes) most = below + step * (f + 1);
        below += step * f;
      }
      lim = max(lim, most - 1);
      if (lim == 0x7fffffffu) --lim;                               // -0's key, which no score has: as a number it is 0 itself
    }
    const double w_tie = cut.ties ? wt(cut_f) : 0.0;
    const unsigned int ties_kept = cut.ties && (enough(w_tie) || cut.key == top_key) ? cut.ties : 0u;
    // sums of the warps' segments of [a, a + len): kept keys are queued so that every lane of the 64-bit arithmetic has one
    auto segments = [&](int a, int len, int seg) {
      double sum = 0.0;
      unsigned int ties = 0, queued = 0;
      float* q = s.queue[warp];
      const int at = min(warp * seg, len), b0 = a + at, b1 = b0 + min(seg, len - at);   // (16 segments can pass 2^31)
      const float lim_f = value_of(lim);
      auto take = [&](float e) {                                   // NaN for lanes without an item
        ties += e == cut_f;
        const bool keep = e > lim_f;
        const unsigned int keeps = __ballot_sync(0xffffffffu, keep);
        if (keep) q[queued + __popc(keeps & ((1u << lane) - 1))] = e;
        queued += __popc(keeps);
        if (queued >= 32) {
          __syncwarp();
          sum += wt(q[lane]);
          const float rest = lane + 32 < queued ? q[lane + 32] : 0.f;
          queued -= 32;
          __syncwarp();
          if (lane < queued) q[lane] = rest;
        }
      };
      // any order does for a sum: lanes read vectors where the segment is aligned
      constexpr int V = 16 / sizeof(T);
      const int head = min(b1 - b0, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x + b0) & 15)) & 15) / static_cast<int>(sizeof(T)));
      const int nv = b1 > b0 ? (b1 - b0 - head) / V : 0, tail = b0 + max(head, 0) + nv * V;
      if (tabled) {
        if constexpr (sizeof(T) == 2) {
          double more = 0.0;
          auto add = [&](uint32_t k, double& to) {
            to += weight16(k >= low16 ? k : 0);                    // (dropped ones all read one zero: no bank is asked twice)
            ties += k == tie16 || k == tie16b;
          };
          auto add2 = [&](uint32_t two) {
            const uint32_t k = patterns_of(two);
            add(k & 0xffffu, sum);
            add(k >> 16, more);
          };
          const unsigned short* xb = reinterpret_cast<const unsigned short*>(x);
          if (lane < head) add(patterns_of(xb[b0 + lane]) & 0xffffu, sum);
          const uint4* xv = reinterpret_cast<const uint4*>(x + b0 + head);
#pragma unroll 2
          for (int i = lane; i < nv; i += 32) {
            const uint4 v = xv[i];
            add2(v.x); add2(v.y); add2(v.z); add2(v.w);
          }
          if (tail + lane < b1) add(patterns_of(xb[tail + lane]) & 0xffffu, sum);
          sum += more;
        }
      } else if (b1 > b0) {
        take(lane < head ? to_f<T>(x[b0 + lane]) : NAN);
        const uint4* xv = reinterpret_cast<const uint4*>(x + b0 + head);
        uint4 next = make_uint4(0, 0, 0, 0);
        if (lane < nv) next = xv[lane];
        for (int i = 0; i < nv; i += 32) {
          const uint4 u = next;
          if (i + 32 + lane < nv) next = xv[i + 32 + lane];
          const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int j = 0; j < V; ++j) take(i + lane < nv ? to_f<T>(e[j]) : NAN);
        }
        take(tail + lane < b1 ? to_f<T>(x[tail + lane]) : NAN);
      }
      __syncwarp();
      if (lane < queued) sum += wt(q[lane]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      ties = __reduce_add_sync(0xffffffffu, ties);
      __syncthreads();
      if (lane == 0) { s.wsum[warp] = sum; s.wcnt[warp] = ties; }
      __syncthreads();
    };
    int a = 0, len = n, seg = ((n + NWARP - 1) / NWARP + 31) / 32 * 32;
    segments(a, len, seg);
    if (tid == 0) {
      double sum = 0.0;
      unsigned int ties = 0;
      for (int i = 0; i < NWARP; ++i) { sum += s.wsum[i]; ties += s.wcnt[i]; }
      s.sum = sum;
      s.ties = ties;
    }
    sync();
    double total = 0.0, before = 0.0, target;
    unsigned int ties_left = ties_kept;
    int owner = -1;
    {
      unsigned int left = ties_kept;
      for (int r = 0; r < c; ++r) {
        const unsigned int t = min(peer(r).ties, left);
        total += peer(r).sum + t * w_tie;
        left -= t;
      }
      target = u * total;
      double run = 0.0;
      left = ties_kept;
      for (int r = 0; r < c; ++r) {
        const unsigned int t = min(peer(r).ties, left);
        const double m = peer(r).sum + t * w_tie;
        if (m > 0.0) {                                             // the last one with any weight, if rounding leaves none
          owner = r; before = run; ties_left = left;
          if (run + m > target) break;
        }
        run += m;
        left -= t;
      }
    }
    if (rank == owner) {
      target -= before;
      for (;;) {
        // every warp walks the sums alike, one per lane
        static_assert(NWARP <= 32, "one sum per lane");
        unsigned int tied = lane < NWARP ? s.wcnt[lane] : 0;
        const unsigned int own_ties = tied;
#pragma unroll
        for (int o = 1; o < NWARP; o <<= 1) {
          const unsigned int y = __shfl_up_sync(0xffffffffu, tied, o);
          if (lane >= o) tied += y;
        }
        const unsigned int used_before = min(tied - own_ties, ties_left);
        const double m = lane < NWARP ? s.wsum[lane] + (min(tied, ties_left) - used_before) * w_tie : 0.0;
        double run = m;
#pragma unroll
        for (int o = 1; o < NWARP; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += y;
        }
        const unsigned int over = __ballot_sync(0xffffffffu, m > 0.0 && run > target), any = __ballot_sync(0xffffffffu, m > 0.0);
        const int pick = over ? __ffs(over) - 1 : 31 - __clz(any);
        const double to_pick = __shfl_sync(0xffffffffu, run, max(pick - 1, 0));
        if (pick > 0) target -= to_pick;
        ties_left -= __shfl_sync(0xffffffffu, used_before, pick);
        len = min(seg, len - pick * seg);
        a += pick * seg;
        if (len <= 32) break;
        seg = ((len + NWARP - 1) / NWARP + 31) / 32 * 32;
        segments(a, len, seg);
      }
      if (warp == 0) {
        const uint32_t k = lane < len ? key_of(to_f<T>(x[a + lane])) : 0u;
        const bool tie = lane < len && k == cut.key;
        const unsigned int tied = __ballot_sync(0xffffffffu, tie);
        double w = 0.0;
        if constexpr (sizeof(T) == 2) {
          if (tabled && lane < len) {
            const uint32_t k16 = patterns_of(reinterpret_cast<const unsigned short*>(x)[a + lane]) & 0xffffu;
            if (k16 >= low16) w = weight16(k16);
          }
        }
        if (!tabled && lane < len && k > lim) w = wk(k);
        if (tie && __popc(tied & ((1u << lane) - 1)) < static_cast<int>(min(ties_left, 32u))) w = w_tie;
        double run = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += v;
        }
        const unsigned int over = __ballot_sync(0xffffffffu, w > 0.0 && run > target), any = __ballot_sync(0xffffffffu, w > 0.0);
        const int pick = over ? __ffs(over) - 1 : 31 - __clz(any);
        if (lane == pick) {
          p.ids[row] = s_lo + a + lane;
          p.logprobs[row] = static_cast<float>(log(w / total));
        }
      }
    }
    sync();                                                        // nobody's words are still being read
  }
}

template <typename T>
int launch(SampleArgs p, int num_sms, cudaStream_t st) {
  constexpr int fixed_bytes = (sizeof(Shared) + 15) / 16 * 16 + 16;
  constexpr int max_bytes = 227 * 1024;
  // The most a row can have (of jagged rows: all but never, so assume twice the average).
  long long longest = p.width;
  if (p.offsets) longest = min(p.width, 2 * p.width / p.rows + 1024);
  // 16-bit scores are counted by one CTA per row, however few rows there are: its fixed part (zeroing, listing and weighing the
  // patterns) is 10 us, its two passes 20 us for 131071 items; by weight it took 17 against 14 us at 1500 items a row, 21 against
  // 15 at 8192, 105 against 40 at 131071, and shared by four CTAs still 46.  Small k are left to the list (256 x 131071, k = 50: 81
  // against 112 us), and the largest score needs no counts.  A k per row is not known here and may be large or 0; where all are
  // small after all, few rows pay for the one CTA (k = 50 as a number / per row: 16 rows 27 / 51 us, 64 rows 33 / 52, 148 55 / 55).
  p.counted = sizeof(T) == 2 && longest > LIST && (p.temperature || p.temperature_v > 0.f) && (p.top_k || p.top_k_v <= 0 || p.top_k_v > LIST / 2);
  // Otherwise CTAs per row: as many as run at once (one per SM: its 16 warps need 128 registers a thread to keep several items'
  // arithmetic in flight), while each keeps some thousand items.  131071 fp32 items with one / two / four CTAs: 114 / 70 /
  // 45 us; 8192: 19 / 20 / 23.  Clusters that do not all run at once cost more than they save: 36 rows by four took 86 us, since
  // clusters of four leave an eighth of the SMs over; of eight, more (16 rows by eight 86 us, by four 44).
  int c = 1;
  auto fits = [&](int by) { return by * p.rows <= (by < 4 ? num_sms : by == 4 ? num_sms - num_sms / 8 : num_sms / 2); };
  if (!p.counted) while (c < MAX_CLUSTER && fits(2 * c) && longest / c > (c < 4 ? 8192 : 65536)) c *= 2;
  const long long slice = (((longest + c - 1) / c + 31) / 32 * 32) * static_cast<long long>(sizeof(T));
  const int count_bytes = p.counted ? COUNT_BYTES : 0;
  const long long room = min(slice, static_cast<long long>(max_bytes - fixed_bytes - count_bytes));
  p.cap = static_cast<int>(room / sizeof(T));
  const int bytes = fixed_bytes + count_bytes + static_cast<int>(room);
  static std::atomic<unsigned long long> done{0};
  const int rc = rb_host::allow_smem(sample_kernel<T>, max_bytes, done);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(c) * static_cast<unsigned>(min(p.rows, 65536)));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = c; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, sample_kernel<T>, p));
}

}  // namespace

// The arguments of rb_sample_scores, 8-byte fields first (packed by the caller).
// scores: fp32 / fp16 / bf16 (dtype 0 / 1 / 2), dense rows of `width` elements `ld` apart, or - with offsets (int32 or int64
// device array [rows + 1]) - jagged in a vector of `width` elements.  uniform [rows] in [0, 1).  Per-row parameters, where
// given, replace the scalar ones: temperature <= 0 takes the largest score, top_k <= 0 and top_p >= 1 are off, min_p is
// relative to the largest weight.  ids [rows] int64 (index within the row, -1: nothing to draw), logprobs [rows]: log of
// the drawn item's share of the kept weights.
struct SampleCall {
  const void* scores; long long ld; const void* offsets; long long width;
  const float *uniform, *temperature; const int* top_k; const float *top_p, *min_p;
  long long* ids; float* logprobs; cudaStream_t stream;
  int offsets64, rows, top_k_v, dtype, num_sms;
  float temperature_v, top_p_v, min_p_v;
};

RB_API int rb_sample_scores(const void* call) {
  const SampleCall& c = *static_cast<const SampleCall*>(call);
  if (c.rows == 0) return 0;
  if (c.width > 0x7fffffffLL - 64) return -1;
  SampleArgs p;
  p.scores = c.scores; p.ld = c.ld; p.offsets = c.offsets; p.offsets64 = c.offsets64; p.width = c.width; p.rows = c.rows; p.cap = 0;
  p.uniform = c.uniform; p.temperature = c.temperature; p.top_k = c.top_k; p.top_p = c.top_p; p.min_p = c.min_p;
  p.temperature_v = c.temperature_v; p.top_k_v = c.top_k_v; p.top_p_v = c.top_p_v; p.min_p_v = c.min_p_v;
  p.ids = c.ids; p.logprobs = c.logprobs;
  const int sms = c.num_sms > 0 ? c.num_sms : 148;
  if (c.dtype == 0) return launch<float>(p, sms, c.stream);
  if (c.dtype == 1) return launch<__half>(p, sms, c.stream);
  if (c.dtype == 2) return launch<__nv_bfloat16>(p, sms, c.stream);
  return -2;
}
