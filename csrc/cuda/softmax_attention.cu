// Softmax attention over the paged KV cache for few query rows per sequence (single tokens, beams), forward (sm_100a).
//
//   o = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q.k_j - max),   lse = max + log sum_j w_j
//
// over the keys that the row sees: up to its own position, of those the last `window` and the first `sinks`.  One pass
// over K and V with a running maximum and sum; both are kept in fp32, as is o.  w is rounded to the inputs' type for the
// product with V (the sum takes it unrounded): a rounding of at most half a step per weight, which averages out over the
// keys to about the rounding of the result itself.  fp16 has no exponents below 2^-14 and nothing below 2^-24, and keys whose
// weights are smaller than that can be many enough to matter, so w is held 2^15 times as large there (`WeightTop`): off by half a step
// down to 2^-29 of the largest weight and by 2^-40 of it below.
//
// Bound: the bytes of K and V.  The G query heads that share a key head are the rows of one 16-row mma.sync tile (a
// 128-row tcgen05 tile would be mostly padding here and the matrix rate does not matter), so K and V are read once for all
// of them.  The keys of all (sequence, row tile, key head) items are laid end to end and every worker takes an equal,
// contiguous share, found from the offsets on the device: uneven histories cost nothing, no length is needed on the host and
// a captured graph stays right for other lengths.  An item cut by a share's border leaves partial results (normalised o
// and its lse) that a second kernel joins.
//
// A worker is one warp where there are enough items to go round - every warp streams its own keys and nothing waits for
// anything else - and a CTA of eight otherwise, whose warps take turns at the tiles of an item and are joined in shared
// memory.  Every warp feeds its own ring by TMA (128-byte swizzle, read with ldmatrix), the page rows of 32 boxes looked up
// at a time.
//
// 128 single tokens of 32 heads over 8 key heads of 128, a window of 4096 and uneven histories: 1.9 GB in 320 us, nine tenths of a
// copy's bandwidth.  Heads of 64 are read in pieces of 128 bytes: 148 sequences of 8000 keys with 8 key heads, where the warps of a
// CTA stand at the same keys of neighbouring heads, reach 6.0 TB/s, 128 such sequences, where they do not, 4.1 (heads of 128: 6.3
// and 6.0).
#include "softmax_attention.cuh"

namespace {

using namespace rb_attn;

constexpr int RT = 16;      // rows per tile
constexpr int NW = 8;       // warps per CTA

template <int D> struct Cfg {
  static constexpr int CH = D / 64;
  static constexpr int KT = 2048 / D;                           // keys per tile
  static constexpr int TILE = KT * D * 2;                       // bytes of a K or a V tile
  static constexpr int STAGES = 3;
  static constexpr int WARP_RING = STAGES * 2 * TILE;
  static constexpr int RING = NW * WARP_RING;
  static constexpr int SMEM = RING + 1024 + 2048;
};

struct Items { int qt, units; };           // row tiles of a sequence, units of W key tiles of each

template <int KT, int W>
__device__ __forceinline__ Items items_of(const Batch& p, const Seq& s) {
  Items r;
  r.qt = (s.len_q * p.G + RT - 1) / RT;
  int tiles;
  if (r.qt <= 1) {
    tiles = span_of<KT>(p, s, 0, max(s.len_q - 1, 0)).tiles;
  } else {                                  // as many for every row tile: the most that one can need
    tiles = (s.len_k + KT - 1) / KT;
    if (s.causal && p.window > 0)
      tiles = static_cast<int>(min(static_cast<long long>(tiles),
                                   (p.sinks + KT - 1LL) / KT + (static_cast<long long>(p.window) + (RT - 1) / p.G + 2 + 2 * KT) / KT));
  }
  r.units = max((tiles + W - 1) / W, 1);
  return r;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}

template <int D, bool BF16, int W>
__global__ void __launch_bounds__(NW * 32, 1) attn_rows_kernel(const __grid_constant__ CUtensorMap tm, const Batch p, const Outs w) {
  using C = Cfg<D>;
  constexpr int KT = C::KT;
  constexpr int PER_CTA = NW / W;                                              // workers of a CTA
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* tail = smem + C::RING;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail);                          // [NW][STAGES]
  long long* sums = reinterpret_cast<long long*>(tail + 256);                  // [NW]
  long long* found_base = reinterpret_cast<long long*>(tail + 320);            // [NW]
  int* found = reinterpret_cast<int*>(tail + 384);                             // [NW]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 416);
  long long* starts = reinterpret_cast<long long*>(tail + 448);                // [NW + 1] where the workers' shares begin
  float* ml = reinterpret_cast<float*>(tail + 1024);                           // [NW][RT][2]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nb = p.a.B + p.b.B;
  launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < NW * C::STAGES; ++i) rb::mbar_init(&bars[i], 1);
    *abort_flag = 0;
    rb::mbar_fence_init();
  }
  // ---- the workers' shares of the keys
  const int per = (nb + NW * 32 - 1) / (NW * 32);
  auto units_of = [&](const Items& it) { return static_cast<long long>(it.qt) * it.units * p.Hkv; };
  long long mine = 0;
  for (int i = tid * per; i < min((tid + 1) * per, nb); ++i) mine += units_of(items_of<KT, W>(p, seq_of(p, i)));
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
  for (int i = 0; i < NW; ++i) {
    if (i < warp) before += sums[i];
    total += sums[i];
  }
  const Shares sh(total, gridDim.x * PER_CTA);
  if (tid <= PER_CTA) {
    const int c = blockIdx.x * PER_CTA + tid;
    starts[tid] = c <= sh.n ? sh.begin(c) : -1;
  }
  __syncthreads();
  // the sequences that the CTA's workers begin with: those of the threads that counted them
  long long last = -1;
#pragma unroll
  for (int x = 0; x < PER_CTA; ++x) if (starts[x + 1] >= 0) last = starts[x];
  if (mine > 0 && starts[0] < before + mine && last >= before) {
    long long base = before;
    for (int i = tid * per; i < min((tid + 1) * per, nb); ++i) {
      const long long n = per == 1 ? mine : units_of(items_of<KT, W>(p, seq_of(p, i)));
#pragma unroll
      for (int x = 0; x < PER_CTA; ++x)
        if (starts[x + 1] >= 0 && starts[x] >= base && starts[x] < base + n) { found[x] = i; found_base[x] = base; }
      base += n;
    }
  }
  __syncthreads();
  const int me = W == 1 ? warp : 0, turn = W == 1 ? 0 : warp;                  // worker of the CTA, this warp's turn in it
  const int wk = blockIdx.x * PER_CTA + me;
  const long long p0 = starts[me + 1] >= 0 ? starts[me] : 0, p1 = max(starts[me + 1], 0LL);
  Meta m;
  m.valid = 0;
  if (p0 < p1) {
    int b = found[me];
    long long base = found_base[me], pos = p0;
    uint8_t* ring = smem + warp * C::WARP_RING;
    uint64_t* bar = bars + warp * C::STAGES;
    int issued = 0, used = 0, st_in = 0, st_out = 0;                           // tiles of this warp so far, ring slots
    uint32_t par = 0;
    bool dead = false;
    const int boxes = KT / p.box_rows, batch = 32 / boxes;
    const int my_kind = lane / (boxes * C::CH), my_box = lane / C::CH % boxes, my_chunk = lane % C::CH;   // this lane's TMA box
    while (pos < p1 && b < nb) {
      const Seq s = seq_of(p, b);
      const Items it = items_of<KT, W>(p, s);
      const long long n_b = units_of(it);
      if (pos >= base + n_b) { base += n_b; ++b; continue; }
      const unsigned long long at = static_cast<unsigned long long>(pos - base);
      const int item = static_cast<int>(at >> 32 ? at / it.units : static_cast<uint32_t>(at) / static_cast<uint32_t>(it.units));
      const int off = static_cast<int>(pos - base - static_cast<long long>(item) * it.units);
      const int qt = item / p.Hkv, h0 = item - qt * p.Hkv;
      const int rows = min(s.len_q * p.G - qt * RT, RT);
      const Span sp = span_of<KT>(p, s, qt * RT / p.G, (qt * RT + rows - 1) / p.G);
      const long long t0 = pos - off;
      if (pos == p0 && off > 0 && sh.begin(wk - 1) <= t0) {
        // the first border inside this item: the second kernel joins its pieces
        m.valid = 1; m.seq = b; m.row0 = qt * RT; m.rows = rows; m.h = h0;
        m.c0 = wk - 1;
        m.c1 = sh.of(t0 + it.units - 1);
        m.first = 2 * m.c0 + (sh.begin(m.c0) == t0 ? 0 : 1);                  // its share's first piece or its last
      }
      // A warp on its own goes through all of its heads of the row tile in one: the ring runs on from one to the next.
      const long long stop = min(p1, W == 1 ? t0 + static_cast<long long>(p.Hkv - h0) * it.units : t0 + it.units);
      const int heads = W == 1 ? static_cast<int>((stop - t0 + it.units - 1) / it.units) : 1;
      const int u_last = static_cast<int>(stop - t0 - static_cast<long long>(heads - 1) * it.units);   // units of the last head
      // key tiles of head h0 + i: begin(i), begin(i) + W, ... below end(i)
      auto begin = [&](int i) { return (i == 0 ? off * W : 0) + turn; };
      auto end = [&](int i) { return min((i == heads - 1 ? u_last : it.units) * W, sp.tiles); };
      int rows_at = -1, rows_box = 0;                                          // rows of the boxes of `batch` tiles from rows_at on
      int in_h = 0, in_v = begin(0);                                           // the next tile to load
      auto issue = [&]() {
        while (in_v >= end(in_h)) {
          if (++in_h >= heads) return;
          in_v = begin(in_h);
        }
        if (rows_at < 0 || in_v < rows_at || in_v >= rows_at + batch * W) {
          rows_at = in_v;
          const int mine_v = in_v + lane / boxes * W;
          rows_box = mine_v < sp.tiles && lane < batch * boxes ? box_row(p, s, sp, sp.tile(mine_v) * KT + (lane % boxes) * p.box_rows) : p.total_rows;
        }
        const int row = __shfl_sync(0xffffffffu, rows_box, ((in_v - rows_at) / W * boxes + my_box) & 31) + my_kind * p.page_size;
        if (lane == 0) rb::mbar_expect_tx(&bar[st_in], 2 * C::TILE);
        __syncwarp();
        if (my_kind < 2)
          rb::tma_load_2d(ring + (st_in * 2 + my_kind) * C::TILE + my_chunk * (KT * 128) + my_box * p.box_rows * 128, &tm, &bar[st_in],
                          (h0 + in_h) * D + my_chunk * 64, row);
        in_v += W;
        ++issued;
        if (++st_in == C::STAGES) st_in = 0;
      };
      if (!dead) for (int i = 0; i < C::STAGES && in_h < heads; ++i) issue();
      // this thread's rows of the 16: lane / 4 and lane / 4 + 8
      bool live[2];
      int rtok[2], rhead[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = (lane >> 2) + 8 * e;
        live[e] = r < rows;
        const int row = qt * RT + (live[e] ? r : 0);
        rtok[e] = row / p.G;
        rhead[e] = row - rtok[e] * p.G;
      }
      for (int ih = 0; ih < heads; ++ih) {
        const int h = h0 + ih;
        // ---- the 16 query rows as A fragments
        uint32_t qf[D / 16][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (s.q_begin + rtok[e]) * p.ld_q +
                                static_cast<long long>(h * p.G + rhead[e]) * D + (lane & 3) * 2;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            qf[kk][e] = live[e] ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16)) : 0u;
            qf[kk][e + 2] = live[e] ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16 + 8)) : 0u;
          }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};               // mx: the maximum less WeightTop
        for (int v = begin(ih); v < end(ih) && !dead; v += W) {
          const bool ok = rb::mbar_wait(&bar[st_out], par, abort_flag, p.status);
          if (!__all_sync(0xffffffffu, ok)) { dead = true; break; }
          ++used;
          const uint32_t k_addr = rb::smem_u32(ring + st_out * 2 * C::TILE), v_addr = k_addr + C::TILE;
          const int j0 = sp.tile(v) * KT;
          const bool full = (s.causal ? j0 + KT - 1 <= sp.p_min : j0 + KT <= sp.hi) &&
                            (!s.causal || p.window <= 0 || j0 > sp.p_max - p.window || j0 + KT <= p.sinks);
          float sc[KT / 8][4];
#pragma unroll
          for (int i = 0; i < KT / 8; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
          // S = Q K^T: ldmatrix x4 = 16 keys x 16 columns
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
            for (int i = 0; i < KT / 16; ++i) {
              const int r = i * 16 + (lane & 7) + ((lane >> 4) << 3);
              const int unit = (kk & 3) * 2 + ((lane >> 3) & 1);
              uint32_t b0, b1, b2, b3;
              ldsm4(k_addr + (kk >> 2) * (KT * 128) + r * 128 + ((unit ^ (r & 7)) << 4), b0, b1, b2, b3);
              mma16816<BF16>(sc[2 * i], qf[kk], b0, b1);
              mma16816<BF16>(sc[2 * i + 1], qf[kk], b2, b3);
            }
          }
          float mn[2] = {-INFINITY, -INFINITY};
          uint32_t seen[2] = {~0u, ~0u};                                       // bit j: the row sees key j0 + (lane & 3) * 2 + j
          if (!full) {
#pragma unroll
            for (int e = 0; e < 2; ++e) seen[e] = seen_keys(rtok[e] + s.delta(), j0, s.len_k, s.causal, p.window, p.sinks) >> ((lane & 3) * 2);
          }
#pragma unroll
          for (int i = 0; i < KT / 8; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = sc[i][e] * p.scale_log2;
              if (!(seen[e >> 1] & (1u << (i * 8 + (e & 1))))) x = -INFINITY;
              sc[i][e] = x;
              mn[e >> 1] = fmaxf(mn[e >> 1], x);
            }
          }
          float corr[2], base_m[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mn[e] = fmaxf(mn[e], __shfl_xor_sync(0xffffffffu, mn[e], 1));
            mn[e] = fmaxf(mn[e], __shfl_xor_sync(0xffffffffu, mn[e], 2));
            mn[e] = fmaxf(mx[e], __fsub_ru(mn[e], WeightTop<BF16>));              // (up: x - mn is never above WeightTop)
            base_m[e] = mn[e] == -INFINITY ? 0.f : mn[e];
            corr[e] = exp2_approx(mx[e] - base_m[e]);
            mx[e] = mn[e];
            sum[e] *= corr[e];
          }
          uint32_t pf[KT / 16][4];
#pragma unroll
          for (int i = 0; i < KT / 8; ++i) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[e] = exp2_approx(sc[i][e] - base_m[e >> 1]);
              sum[e >> 1] += x[e];
            }
            pf[i >> 1][(i & 1) * 2] = pack16<BF16>(x[0], x[1]);
            pf[i >> 1][(i & 1) * 2 + 1] = pack16<BF16>(x[2], x[3]);
          }
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1];
          }
          if (!(j0 + KT <= sp.hi && (j0 >= sp.lo || j0 + KT <= sp.sinks))) {
            // V of keys that no row of the block sees may be anything (0 x NaN is NaN): clear it
            const int j = j0 + lane;
            if (lane < KT && !(j < sp.hi && (j >= sp.lo || j < sp.sinks))) {
              uint4* vr = reinterpret_cast<uint4*>(ring + (st_out * 2 + 1) * C::TILE + lane * 128);
#pragma unroll
              for (int c = 0; c < C::CH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) vr[c * (KT * 8) + ((i + lane) & 7)] = make_uint4(0, 0, 0, 0);
            }
            rb::fence_proxy_async_smem();
            __syncwarp();
          }
          // O += P V
#pragma unroll
          for (int kk = 0; kk < KT / 16; ++kk) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              const int r = kk * 16 + (lane & 15);
              const int unit = (i & 3) * 2 + (lane >> 4);
              uint32_t b0, b1, b2, b3;
              ldsm4_trans(v_addr + (i >> 2) * (KT * 128) + r * 128 + ((unit ^ (r & 7)) << 4), b0, b1, b2, b3);
              mma16816<BF16>(o[2 * i], pf[kk], b0, b1);
              mma16816<BF16>(o[2 * i + 1], pf[kk], b2, b3);
            }
          }
          __syncwarp();
          if (++st_out == C::STAGES) { st_out = 0; par ^= 1; }
          if (in_h < heads) issue();
        }
        if (dead) {                                                              // the kernel's own copies end before it does
          for (; used < issued; ++used) {
            for (uint32_t i = 0; i < (1u << 20) && !rb::mbar_try_wait(&bar[st_out], par); ++i) {}
            if (++st_out == C::STAGES) { st_out = 0; par ^= 1; }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
          sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
        }
        const bool whole = (ih > 0 || off == 0) && (ih < heads - 1 || u_last == it.units);
        const long long cut = static_cast<long long>(wk) * 2 + (pos == p0 && ih == 0 ? 0 : 1);
        if (W == 1) {
          // ---- the warp's own result, straight from the fragments
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = (lane >> 2) + 8 * e;
            if (live[e]) {
              const float inv = sum[e] == 0.f ? 0.f : 1.f / sum[e];
              const float lse2 = sum[e] == 0.f ? -INFINITY : mx[e] + log2f(sum[e]);
              const RowOut to = row_out(p, w, s, qt * RT + r, h, D, whole, cut * RT + r);
              if ((lane & 3) == 0 && to.lse) *to.lse = to.natural ? lse2 * LN2 : lse2;
#pragma unroll
              for (int i = 0; i < D / 8; ++i) {
                const float x = o[i][2 * e] * inv, y = o[i][2 * e + 1] * inv;
                const int col = i * 8 + (lane & 3) * 2;
                if (to.o16) *reinterpret_cast<uint32_t*>(to.o16 + col) = pack16<BF16>(x, y);
                else *reinterpret_cast<float2*>(to.o32 + col) = make_float2(x, y);
              }
            }
          }
        } else {
          // ---- join the warps: o [RT][D] in the warp's own, now idle ring
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = (lane >> 2) + 8 * e;
            float* dst = reinterpret_cast<float*>(ring) + r * D + (lane & 3) * 2;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
            if ((lane & 3) == 0) { ml[(warp * RT + r) * 2] = mx[e]; ml[(warp * RT + r) * 2 + 1] = sum[e]; }
          }
          __syncthreads();
          constexpr int TPR = NW * 32 / RT, N = 4;                               // threads per row, elements at a time
          const int r = tid / TPR;
          if (r < rows) {
            float mm = -INFINITY;
#pragma unroll
            for (int i = 0; i < NW; ++i) mm = fmaxf(mm, ml[(i * RT + r) * 2]);
            const float bm = mm == -INFINITY ? 0.f : mm;
            float f[NW], l = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
              f[i] = exp2_approx(ml[(i * RT + r) * 2] - bm);
              l += f[i] * ml[(i * RT + r) * 2 + 1];
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const float lse2 = l == 0.f ? -INFINITY : mm + log2f(l);
            const RowOut to = row_out(p, w, s, qt * RT + r, h, D, whole, cut * RT + r);
            if (tid % TPR == 0 && to.lse) *to.lse = to.natural ? lse2 * LN2 : lse2;
            for (int col = (tid % TPR) * N; col < D; col += TPR * N) {
              float x[N] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int i = 0; i < NW; ++i) {
                const float4 y = *reinterpret_cast<const float4*>(smem + i * C::WARP_RING + (r * D + col) * 4);
                x[0] += f[i] * y.x; x[1] += f[i] * y.y; x[2] += f[i] * y.z; x[3] += f[i] * y.w;
              }
              if (to.o16) *reinterpret_cast<uint2*>(to.o16 + col) = make_uint2(pack16<BF16>(x[0] * inv, x[1] * inv), pack16<BF16>(x[2] * inv, x[3] * inv));
              else *reinterpret_cast<float4*>(to.o32 + col) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
            }
          }
          rb::fence_proxy_async_smem();
          __syncthreads();
        }
      }
      pos = stop;
    }
  }
  if (lane == 0 && (W == 1 || warp == 0)) w.meta[wk] = m;
  if (tid == 0) wait_before();                                                 // what ran before is done when this kernel is
}

// One kernel's cut items, `split` blocks for each share; a call has those of the rows kernel, of the tiles kernel or of both.
struct Join { Batch p; Outs w; int shares, split, block_rows; };
struct Joins { Join of[2]; };

// Joins the pieces of the items that borders cut: a share's blocks look after the item whose first border is its begin,
// 16 rows at a time and four columns per thread.  Items have up to `block_rows` rows.  (Few blocks: most of them find nothing to
// do, and it is their number that this kernel's time goes by.)
template <int D, bool BF16>
__global__ void __launch_bounds__(RT * D / 4) attn_join_kernel(const __grid_constant__ Joins j) {
  launch_dependents();
  wait_before();
  const bool second = static_cast<int>(blockIdx.x) >= j.of[0].shares * j.of[0].split;
  const Join& of = j.of[second];
  const int b = blockIdx.x - (second ? j.of[0].shares * j.of[0].split : 0), block_rows = of.block_rows;
  const Batch& p = of.p;
  const Outs& w = of.w;
  const Meta m = w.meta[b / of.split];
  if (!m.valid) return;
  constexpr int STEP = 8;                                                      // pieces in flight
  const int col = threadIdx.x % (D / 4) * 4;
  const Seq s = seq_of(p, m.seq);
  for (int r = b % of.split * RT + threadIdx.x / (D / 4); r < m.rows; r += of.split * RT) {
    auto place = [&](int c) { return static_cast<long long>(c == m.c0 ? m.first : 2 * c) * block_rows + r; };
    float mm = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = m.c0; c <= m.c1; c += STEP) {
      float lse[STEP];
      float4 y[STEP];
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        lse[i] = -INFINITY;
        y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c + i <= m.c1) {
          const long long at = place(c + i);
          lse[i] = w.cut_lse[at];
          y[i] = *reinterpret_cast<const float4*>(w.cut_o + at * D + col);
        }
      }
      float top = mm;
#pragma unroll
      for (int i = 0; i < STEP; ++i) top = fmaxf(top, lse[i]);
      const float bm = top == -INFINITY ? 0.f : top, f0 = exp2_approx(mm - bm);
      mm = top;
      l *= f0;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] *= f0;
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        const float f = exp2_approx(lse[i] - bm);
        l += f;
        x[0] += f * y[i].x; x[1] += f * y[i].y; x[2] += f * y[i].z; x[3] += f * y[i].w;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const float lse2 = l == 0.f ? -INFINITY : mm + log2f(l);
    const RowOut to = row_out(p, w, s, m.row0 + r, m.h, D, true, 0);
    if (col == 0 && to.lse) *to.lse = to.natural ? lse2 * LN2 : lse2;
    if (to.o16) *reinterpret_cast<uint2*>(to.o16 + col) = make_uint2(pack16<BF16>(x[0] * inv, x[1] * inv), pack16<BF16>(x[2] * inv, x[3] * inv));
    else *reinterpret_cast<float4*>(to.o32 + col) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  }
}

// out = the two parts of every row (prefix, suffix), weighted by their sums
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attn_merge_kernel(const Batch p, const Outs w) {
  wait_before();
  constexpr int TPR = D / 4;
  const long long rows = static_cast<long long>(p.Tq) * p.H;
  const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / TPR;
  if (row >= rows) return;
  const int col = (threadIdx.x % TPR) * 4;
  // tokens of requests in no group have no first part, tokens of no request neither
  const int t = static_cast<int>(row / p.H);
  const int* go = p.a.group_offsets;
  const bool has_a = t >= p.a.q_offsets[go ? min(max(go[0], 0), p.a.num_requests) : 0] &&
                     t < p.a.q_offsets[go ? min(max(go[p.a.B], 0), p.a.num_requests) : p.a.num_requests];
  const bool has_b = t >= p.b.q_offsets[0] && t < p.b.q_offsets[p.b.B];
  const float a = has_a ? w.part_lse[row] : -INFINITY, b = has_b ? w.part_lse[rows + row] : -INFINITY;
  const float mm = fmaxf(a, b), bm = mm == -INFINITY ? 0.f : mm;
  const float fa = exp2_approx(a - bm), fb = exp2_approx(b - bm), l = fa + fb;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
  if (has_a) x = *reinterpret_cast<const float4*>(w.part_o + row * D + col);
  if (has_b) y = *reinterpret_cast<const float4*>(w.part_o + (rows + row) * D + col);
  const float z0 = (fa * x.x + fb * y.x) * inv, z1 = (fa * x.y + fb * y.y) * inv, z2 = (fa * x.z + fb * y.z) * inv,
              z3 = (fa * x.w + fb * y.w) * inv;
  uint16_t* dst = reinterpret_cast<uint16_t*>(w.out) + t * w.ld_o + (row % p.H) * D + col;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<BF16>(z0, z1), pack16<BF16>(z2, z3));
  if (col == 0 && w.lse) w.lse[row] = l == 0.f ? -INFINITY : (mm + log2f(l)) * LN2;
}

constexpr long long align256(long long n) { return (n + 255) / 256 * 256; }

// Workspace: the pieces of the rows kernel, those of the tiles kernel, the two parts of rows behind a prefix.
struct Space { long long cut_o[2], cut_lse[2], meta[2], part_o, part_lse, total; };

Space space_of(int n_cta, int D, long long rows, bool with_rows, bool with_tiles, bool parts) {
  Space s;
  long long at = 0;
  auto take = [&](long long bytes) { const long long was = at; at = align256(at + bytes); return was; };
  for (int k = 0; k < 2; ++k) {
    const long long n = (k ? with_tiles : with_rows) ? static_cast<long long>(n_cta) * (k ? 1 : NW) : 0, block = k ? TILE_ROWS : RT;
    s.cut_o[k] = take(n * 2 * block * D * 4);
    s.cut_lse[k] = take(n * 2 * block * 4);
    s.meta[k] = take(n * static_cast<long long>(sizeof(Meta)));
  }
  s.part_o = take(parts ? 2 * rows * D * 4 : 0);
  s.part_lse = take(parts ? 2 * rows * 4 : 0);
  s.total = at;
  return s;
}

// Which kernel a list of sequences takes, by the average number of rows that share a key head: the rows kernel reads
// K and V once for 16 of them, the tiles kernel once for 256 with at least 128 computed.  Heads of 128, 32 sequences of 4000
// keys, 16 / 24 / 48 / 128 rows: by rows 96 / 177 / 234 / 626 us, by tiles 98 / 101 / 102 / 111; heads of 64, 200 sequences
// of 1000 keys, 16 / 32 / 48 / 64 rows: by rows 118 / 116 / 153 / 230 us, by tiles 132 / 132 / 133 / 133.  Uneven batches go by the average, too: a
// prompt of 2000 among 200 single tokens over 1000 / 4000 keys, 8 heads of 64, by rows 135 / 426 us, by tiles 164 / 410; among 64 of
// them, 32 heads over 8 of 128, by rows 483 / 565 us, by tiles (which the average takes) 117 / 223.
bool by_tiles(long long Tq, int G, int D, int sequences, float scale) {
  return G <= 128 && scale > 0.f && sequences > 0 && Tq * G * D > 2048LL * sequences;
}

struct Plan { bool tiles_a, tiles_b; };

Plan plan_of(long long Tq, int G, int D, int B, int groups, float scale) {
  const bool own = by_tiles(Tq, G, D, B, scale);
  Plan r;
  r.tiles_a = groups > 0 ? by_tiles(Tq, G, D, groups, scale) : own;
  r.tiles_b = groups > 0 && own;
  return r;
}

template <int D, bool BF16, int W>
int launch_rows(const CUtensorMap& tm, const Batch& p, const Outs& w, int n_cta, bool after, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const int rc = rb_host::allow_smem(attn_rows_kernel<D, BF16, W>, Cfg<D>::SMEM, done);
  if (rc) return rc;
  return launch_kernel(after, attn_rows_kernel<D, BF16, W>, dim3(n_cta), dim3(NW * 32), Cfg<D>::SMEM, st, tm, p, w);
}

template <int D, bool BF16>
int launch(const Batch& p, Outs w, const Plan& plan, const Space& sp, char* ws, const void* cache, int n_cta, cudaStream_t st) {
  const bool parts = p.b.B > 0;
  bool after = false;
  Joins joins = {};
  for (int tiles = 0; tiles < 2; ++tiles) {
    Batch q = p;
    if (plan.tiles_a != (tiles != 0)) q.a.B = 0;
    if (plan.tiles_b != (tiles != 0)) q.b.B = 0;
    if (q.a.B + q.b.B == 0) continue;
    w.cut_o = reinterpret_cast<float*>(ws + sp.cut_o[tiles]);
    w.cut_lse = reinterpret_cast<float*>(ws + sp.cut_lse[tiles]);
    w.meta = reinterpret_cast<Meta*>(ws + sp.meta[tiles]);
    int shares = n_cta;
    if (tiles) {
      const int rc = launch_tiles(q, w, cache, D, BF16, n_cta, after, st);
      if (rc) return rc;
    } else {
      CUtensorMap tm;
      q.box_rows = p.page_size % Cfg<D>::KT == 0 ? Cfg<D>::KT : 16;
      int rc = rb_host::make_map_2d(&tm, cache, p.total_rows, static_cast<long long>(p.Hkv) * D, static_cast<long long>(p.Hkv) * D, 64,
                                    q.box_rows, BF16);
      if (rc) return rc;
      // a worker per warp where there are more items (at least one per sequence and key head) than CTAs.  8000 keys each, heads of
      // 64, 128 / 192 / 1184 items: by warps 63 / 85 / 390 us, by CTAs 52 / 95 / 564; 100 keys: 9.9 / 10.2 / 12.9 and 8.1 / 11.2 /
      // 30.1; heads of 128, 8000 keys: 96 / 138 / 779 and 93 / 135 / 782.
      const bool single = static_cast<long long>(q.a.B + q.b.B) * p.Hkv > n_cta;
      if (single) shares = n_cta * NW;
      rc = single ? launch_rows<D, BF16, 1>(tm, q, w, n_cta, after, st) : launch_rows<D, BF16, NW>(tm, q, w, n_cta, after, st);
      if (rc) return rc;
    }
    joins.of[after] = {q, w, shares, tiles ? 8 : 1, tiles ? TILE_ROWS : RT};
    if (!after) joins.of[1].split = 1;
    after = true;
  }
  if (!after) return 0;
  const int rc = launch_kernel(true, attn_join_kernel<D, BF16>, dim3(joins.of[0].shares * joins.of[0].split + joins.of[1].shares * joins.of[1].split),
                               dim3(RT * D / 4), 0, st, joins);
  if (rc) return rc;
  if (parts) {
    const long long rows = static_cast<long long>(p.Tq) * p.H;
    const int per = 256 / (D / 4);
    const int rc = launch_kernel(true, attn_merge_kernel<D, BF16>, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), 0, st, p, w);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace

// Bytes of workspace that rb_softmax_attn_paged needs.
RB_API long long rb_softmax_attn_workspace(int num_sms, long long Tq, int H, int Hkv, int D, int B, int groups, float scale) {
  if (Hkv <= 0 || H % Hkv) return 0;
  const Plan plan = plan_of(Tq, H / Hkv, D, B, groups, scale);
  return space_of(num_sms > 0 ? num_sms : 148, D, Tq * H, !plan.tiles_a || (groups > 0 && !plan.tiles_b), plan.tiles_a || plan.tiles_b,
                  groups > 0).total;
}

// How many kernels it launches.
RB_API int rb_softmax_attn_kernels(long long Tq, int H, int Hkv, int D, int B, int groups, float scale) {
  if (Tq == 0 || B == 0 || Hkv <= 0 || H % Hkv) return 0;
  const Plan plan = plan_of(Tq, H / Hkv, D, B, groups, scale);
  return 2 + (groups > 0 ? 1 + (plan.tiles_a != plan.tiles_b) : 0);            // rows or tiles or both, join, merge
}

// The arguments of rb_softmax_attn_paged, 8-byte fields first (the caller packs them: by far cheaper than 33 arguments).
// q [Tq][H][D] (token stride ld_q), cache [num_pages][2][page_size][Hkv][D], bf16 or fp16; int32 offsets and page tables on
// the device.  B requests own the queries q_offsets[b]..q_offsets[b+1] and k_offsets[b+1] - k_offsets[b] keys, the last of which are
// the queries' own.  G groups (0: none) of requests group_offsets[g]..group_offsets[g+1] - or, without group_offsets, ONE
// group of all requests - see prefix_offsets[g+1] - prefix_offsets[g] more keys in front of their own; window and sinks
// are for calls without groups.  out [Tq][H][D] (token stride ld_o), lse [Tq][H] fp32 or null.
struct SoftmaxAttnCall {
  const void* q; long long ld_q, Tq;
  const void* cache; long long num_pages;
  const int *q_offsets, *k_offsets, *page_ids, *page_indptr;
  const int *group_offsets, *prefix_offsets, *prefix_page_ids, *prefix_page_indptr;
  void* out; long long ld_o; float* lse;
  void* workspace; long long workspace_bytes;
  int* status; cudaStream_t stream;
  int H, Hkv, D, page_size, num_page_ids, B, num_prefix_page_ids, groups, window, sinks, is_bf16, num_sms;
  float scale;
};

RB_API int rb_softmax_attn_paged(const void* call) {
  const SoftmaxAttnCall& c = *static_cast<const SoftmaxAttnCall*>(call);
  if (c.Tq == 0 || c.B == 0) return 0;
  if ((c.D != 64 && c.D != 128) || c.Hkv <= 0 || c.H % c.Hkv) return -1;
  if (c.ld_q % 8 || c.ld_o % 16) return -2;
  if (c.page_size % 16 || c.page_size <= 0 || (c.groups > 0 && c.window > 0) || (c.groups > 1 && !c.group_offsets)) return -3;
  const long long rows = c.num_pages * 2 * c.page_size;
  if (c.Tq * c.H > 0x7fffffffLL || rows + c.page_size > 0x7fffffffLL) return -4;
  const int n_cta = c.num_sms > 0 ? c.num_sms : 148;
  const Plan plan = plan_of(c.Tq, c.H / c.Hkv, c.D, c.B, c.groups, c.scale);
  const Space sp = space_of(n_cta, c.D, c.Tq * c.H, !plan.tiles_a || (c.groups > 0 && !plan.tiles_b), plan.tiles_a || plan.tiles_b, c.groups > 0);
  if (c.workspace_bytes < sp.total) return -5;
  Batch p;
  const Seqs own = {c.q_offsets, nullptr, 0, c.k_offsets, c.page_ids, c.page_indptr, c.num_page_ids, c.B, c.B, 1};
  const Seqs none = {nullptr, nullptr, 0, nullptr, nullptr, nullptr, 0, 0, 0, 0};
  const Seqs pre = {c.q_offsets, c.group_offsets, c.group_offsets == nullptr, c.prefix_offsets, c.prefix_page_ids, c.prefix_page_indptr,
                    c.num_prefix_page_ids, c.groups, c.B, 0};
  p.a = c.groups > 0 ? pre : own;
  p.b = c.groups > 0 ? own : none;
  p.q = c.q; p.ld_q = c.ld_q; p.Tq = static_cast<int>(c.Tq); p.H = c.H; p.Hkv = c.Hkv; p.G = c.H / c.Hkv; p.page_size = c.page_size;
  p.box_rows = 16; p.total_rows = static_cast<int>(rows); p.window = c.window; p.sinks = c.sinks;
  p.scale_log2 = c.scale * LOG2E; p.status = c.status;
  char* ws = static_cast<char*>(c.workspace);
  Outs w;
  w.out = c.out; w.ld_o = c.ld_o; w.lse = c.lse;
  w.part_o = c.groups > 0 ? reinterpret_cast<float*>(ws + sp.part_o) : nullptr;
  w.part_lse = reinterpret_cast<float*>(ws + sp.part_lse);
  if (c.D == 64)
    return c.is_bf16 ? launch<64, true>(p, w, plan, sp, ws, c.cache, n_cta, c.stream) : launch<64, false>(p, w, plan, sp, ws, c.cache, n_cta, c.stream);
  return c.is_bf16 ? launch<128, true>(p, w, plan, sp, ws, c.cache, n_cta, c.stream) : launch<128, false>(p, w, plan, sp, ws, c.cache, n_cta, c.stream);
}
