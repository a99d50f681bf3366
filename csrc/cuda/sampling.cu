// Drawing one item per row from its scores (sm_100a): temperature, top-k, top-p, min-p, one given uniform number per row.
//
//   w_i = exp((x_i - max) / T);  in the order (score descending, index ascending) keep
//     the first k;  of those, up to the first whose running sum reaches p times their sum;  of those, w_i >= min_p
//   -> the smallest index i whose running sum over the kept items, in index order, exceeds u times their sum.
//
// Every filter keeps a beginning of the same order, so no sort is needed: a radix descent over the 32 ordered bits of the
// score finds the last kept value (by count for k, by weight for p) and how many of the items that share it are kept.
//
// Weights are summed in 64 bits: with 10^5 items of similar score the borders lie 1e-5 apart, and 32-bit exponentials
// (relative error 1e-7 each) would draw a neighbour every few thousand rows.  Sums inside the descent are whole numbers
// (2^-44 of the largest weight for rows up to 2^18 items, coarser beyond), so atomics in any order give the same bits.
#include "common.cuh"

namespace {

constexpr int NT = 512, NWARP = NT / 32;
constexpr int BINS = 2048;

struct SampleArgs {
  const void* scores; long long ld;             // dense: rows of `width`, `ld` elements apart
  const void* offsets; int offsets64;           // jagged: [rows + 1] into scores (then `width` is its length), or null
  long long width; int rows;
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

struct Shared {
  unsigned int cnt[BINS];
  unsigned long long mass[BINS];
  double wsum[NWARP];
  unsigned int wcnt[NWARP];
  unsigned long long wmass[NWARP];
  double d0, d1;
  unsigned long long m0;
  unsigned int u0, u1, u2;
};

// weight of a score
struct Weigher {
  double top, inv_t;
  uint32_t top_key;
  __device__ __forceinline__ double operator()(uint32_t k) const {
    return k == top_key ? 1.0 : exp((static_cast<double>(value_of(k)) - top) * inv_t);
  }
};

// Where the order is cut: everything above `key` is kept and the first `ties` items (in index order) that equal it.
struct Cut { uint32_t key; unsigned int ties; };

template <typename T>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleArgs p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
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
    const int n = static_cast<int>(hi - lo);
    const float temp = p.temperature ? p.temperature[row] : p.temperature_v;
    const int top_k = p.top_k ? p.top_k[row] : p.top_k_v;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_v;
    const float min_p = p.min_p ? p.min_p[row] : p.min_p_v;
    float uf = p.uniform[row];
    const double u = uf > 0.f ? static_cast<double>(uf) : 0.0;
    // ---- the largest score and its first index
    unsigned long long best = 0;                                   // key, then index from the back
    for (int i = tid; i < n; i += NT) {
      const unsigned long long v = (static_cast<unsigned long long>(key_of(to_f<T>(x[i]))) << 32) | (0xffffffffu - i);
      best = v > best ? v : best;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long v = __shfl_xor_sync(0xffffffffu, best, o);
      best = v > best ? v : best;
    }
    __syncthreads();                                               // the row before is done with the shared words
    if (lane == 0) s.wmass[warp] = best;
    __syncthreads();
    for (int i = 0; i < NWARP; ++i) best = s.wmass[i] > best ? s.wmass[i] : best;
    const uint32_t top_key = static_cast<uint32_t>(best >> 32);
    if (n == 0 || top_key <= KEY_NONE) {
      if (tid == 0) { p.ids[row] = -1; p.logprobs[row] = -INFINITY; }
      continue;
    }
    if (!(temp > 0.f)) {
      if (tid == 0) { p.ids[row] = 0xffffffffu - static_cast<uint32_t>(best); p.logprobs[row] = 0.f; }
      continue;
    }
    Weigher wt;
    wt.top = static_cast<double>(value_of(top_key)); wt.inv_t = 1.0 / static_cast<double>(temp); wt.top_key = top_key;
    Cut cut = {KEY_NONE, 0};
    // ---- radix descent: by count, then by weight
    const int shift_fx = 62 - max(18, 32 - __clz(n));
    const double fx = static_cast<double>(1ULL << shift_fx);
    for (int by_mass = 0; by_mass < 2; ++by_mass) {
      if (by_mass ? !(top_p < 1.f) : !(top_k > 0 && top_k < n)) continue;
      uint32_t prefix = 0;
      int bits = 0;
      unsigned int c_before = 0;
      unsigned long long m_before = 0, target = 0;
      bool none = false;
      for (int level = 0; level < 3 && !none; ++level) {
        const int width = level < 2 ? 11 : 10, down = 32 - bits - width;
        for (int i = tid; i < BINS; i += NT) { s.cnt[i] = 0; s.mass[i] = 0; }
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
          const uint32_t k = key_of(to_f<T>(x[i]));
          if (k <= cut.key || (bits && (k >> (32 - bits)) != prefix)) continue;
          const int bin = (k >> down) & ((1 << width) - 1);
          if (by_mass) atomicAdd(&s.mass[bin], static_cast<unsigned long long>(wt(k) * fx + 0.5));
          else atomicAdd(&s.cnt[bin], 1u);
        }
        if (by_mass && tid == 0 && cut.ties && (!bits || (cut.key >> (32 - bits)) == prefix))
          atomicAdd(&s.mass[(cut.key >> down) & ((1 << width) - 1)], cut.ties * static_cast<unsigned long long>(wt(cut.key) * fx + 0.5));
        __syncthreads();
        // the bin where the running sum from above reaches the target: 4 bins per thread, from the highest down
        constexpr int PB = BINS / NT;
        unsigned int c4 = 0;
        unsigned long long m4 = 0;
        for (int i = 0; i < PB; ++i) {
          const int b = BINS - 1 - (tid * PB + i);
          c4 += s.cnt[b];
          m4 += s.mass[b];
        }
        unsigned int ci = c4;
        unsigned long long mi = m4;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned int a = __shfl_up_sync(0xffffffffu, ci, o);
          const unsigned long long b = __shfl_up_sync(0xffffffffu, mi, o);
          if (lane >= o) { ci += a; mi += b; }
        }
        if (lane == 31) { s.wcnt[warp] = ci; s.wmass[warp] = mi; }
        if (tid == 0) s.u2 = 0;
        __syncthreads();
        unsigned int cb = ci - c4, call = 0;
        unsigned long long mb = mi - m4, mall = 0;
        for (int i = 0; i < NWARP; ++i) {
          if (i < warp) { cb += s.wcnt[i]; mb += s.wmass[i]; }
          call += s.wcnt[i];
          mall += s.wmass[i];
        }
        if (level == 0) {
          if (by_mass) {
            const double t = ceil(static_cast<double>(top_p) * static_cast<double>(mall));
            target = t > 1.0 ? static_cast<unsigned long long>(t) : 1ULL;     // at least the first item
          } else {
            none = call <= static_cast<unsigned int>(top_k);                  // fewer items than k: all are kept
          }
        }
        cb += c_before;
        mb += m_before;
        for (int i = 0; i < PB; ++i) {
          const int b = BINS - 1 - (tid * PB + i);
          const bool here = by_mass ? (mb < target && mb + s.mass[b] >= target)
                                    : (cb < static_cast<unsigned int>(top_k) && cb + s.cnt[b] >= static_cast<unsigned int>(top_k));
          if (here) { s.u0 = b; s.u1 = cb; s.m0 = mb; s.u2 = 1; }
          cb += s.cnt[b];
          mb += s.mass[b];
        }
        __syncthreads();
        if (!s.u2) none = true;
        if (!none) {
          prefix = (prefix << width) | s.u0;
          bits += width;
          c_before = s.u1;
          m_before = s.m0;
        }
        __syncthreads();
      }
      if (none) continue;
      if (by_mass) {
        const unsigned long long w = static_cast<unsigned long long>(wt(prefix) * fx + 0.5);
        const unsigned long long r = w ? (target - m_before + w - 1) / w : 0xffffffffULL;
        const unsigned int most = prefix == cut.key ? cut.ties : 0xffffffffu;
        cut.ties = static_cast<unsigned int>(min(r, static_cast<unsigned long long>(most)));
      } else {
        cut.ties = static_cast<unsigned int>(top_k) - c_before;
      }
      cut.key = prefix;
    }
    // ---- draw: split the range among the warps, find the one where the running sum passes u * total, repeat inside it
    const double mp = static_cast<double>(min_p);
    const double w_tie = cut.ties ? wt(cut.key) : 0.0;
    const bool tie_ok = w_tie >= mp || cut.key == top_key;
    auto weight = [&](uint32_t k) -> double {
      if (k <= cut.key) return 0.0;
      const double w = wt(k);
      return w >= mp || k == top_key ? w : 0.0;
    };
    int a = 0, len = n;
    unsigned int ties_left = tie_ok ? cut.ties : 0u;
    double target = 0.0, total = 0.0;
    bool first = true;
    while (first || len > 32) {
      const int seg = ((len + NWARP - 1) / NWARP + 31) / 32 * 32;
      double sum = 0.0;
      unsigned int ties = 0;
      const int b0 = a + warp * seg, b1 = min(b0 + seg, a + len);
      for (int i = b0 + lane; i < b1; i += 32) {
        const uint32_t k = key_of(to_f<T>(x[i]));
        sum += weight(k);
        ties += k == cut.key;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        ties += __shfl_xor_sync(0xffffffffu, ties, o);
      }
      __syncthreads();
      if (lane == 0) { s.wsum[warp] = sum; s.wcnt[warp] = ties; }
      __syncthreads();
      // every thread walks the 16 sums alike
      if (first) {
        unsigned int left = ties_left;
        for (int i = 0; i < NWARP; ++i) {
          const unsigned int t = min(s.wcnt[i], left);
          total += s.wsum[i] + t * w_tie;
          left -= t;
        }
        target = u * total;
        first = false;
      }
      double run = 0.0, pick_run = 0.0;
      unsigned int left = ties_left, pick_left = 0;
      int pick = -1;
      for (int i = 0; i < NWARP; ++i) {
        const unsigned int t = min(s.wcnt[i], left);
        const double m = s.wsum[i] + t * w_tie;
        if (m > 0.0) {                                             // the last one with any weight, if rounding leaves none
          pick = i; pick_run = run; pick_left = left;
          if (run + m > target) break;
        }
        run += m;
        left -= t;
      }
      if (pick < 0) pick = 0;
      target -= pick_run;
      ties_left = pick_left;
      len = min(seg, a + len - (a + pick * seg));
      a += pick * seg;
    }
    if (warp == 0) {
      const int i = a + lane;
      const uint32_t k = lane < len ? key_of(to_f<T>(x[i])) : 0u;
      const bool tie = lane < len && k == cut.key;
      const unsigned int tied = __ballot_sync(0xffffffffu, tie);
      double w = lane < len ? weight(k) : 0.0;
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
        p.ids[row] = i;
        p.logprobs[row] = static_cast<float>(log(w / total));
      }
    }
  }
}

}  // namespace

// scores: fp32 / fp16 / bf16 (dtype 0 / 1 / 2), dense rows of `width` elements `ld` apart, or - with offsets (int32 or int64
// device array [rows + 1]) - jagged in a vector of `width` elements.  uniform [rows] in [0, 1).  Per-row parameters, where
// given, replace the scalar ones: temperature <= 0 takes the largest score, top_k <= 0 and top_p >= 1 are off, min_p is
// relative to the largest weight.  ids [rows] int64 (index within the row, -1: nothing to draw), logprobs [rows]: log of
// the drawn item's share of the kept weights.
RB_API int rb_sample_scores(const void* scores, long long ld, const void* offsets, int offsets64, long long width, int rows,
                            const float* uniform, const float* temperature, const int* top_k, const float* top_p,
                            const float* min_p, float temperature_v, int top_k_v, float top_p_v, float min_p_v, long long* ids,
                            float* logprobs, int dtype, cudaStream_t st) {
  if (rows == 0) return 0;
  if (width > 0x7fffffffLL) return -1;
  SampleArgs p;
  p.scores = scores; p.ld = ld; p.offsets = offsets; p.offsets64 = offsets64; p.width = width; p.rows = rows;
  p.uniform = uniform; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.temperature_v = temperature_v; p.top_k_v = top_k_v; p.top_p_v = top_p_v; p.min_p_v = min_p_v;
  p.ids = ids; p.logprobs = logprobs;
  const int grid = rows < 65536 ? rows : 65536;
  if (dtype == 0) sample_kernel<float><<<grid, NT, 0, st>>>(p);
  else if (dtype == 1) sample_kernel<__half><<<grid, NT, 0, st>>>(p);
  else if (dtype == 2) sample_kernel<__nv_bfloat16><<<grid, NT, 0, st>>>(p);
  else return -2;
  return static_cast<int>(cudaGetLastError());
}
