// Softmax attention over the paged KV cache for many query rows per sequence (prompts, new tokens over a long history, a
// group of requests behind a common prefix), forward, on tcgen05 / TMEM (sm_100a).  The mathematics is that of
// softmax_attention.cu: one pass over K and V with a running maximum and sum in fp32.
//
// Bound: the matrix rate and, equally, the exponentials: 128 rows of a key tile of 64 cost 2 x 128 x 64 x D multiply-adds
// (512 cycles of the tensor core for D = 128) and 8192 exponentials (512 cycles of the special function units).  So two row
// tiles are always in flight, one in the tensor core while the other is in the softmax warps:
//   * 256 rows (two row tiles of 128: 128 / G tokens x the G query heads that share a key head) walk the same key tiles, or
//   * where a block has 128 rows or fewer, one row tile takes even key tiles with one set of warps and odd ones with
//     the other; the two results are joined from TMEM at the end.
// Roles: warp 0 issues TMA loads (Q once per block, then a K and a V tile a slot through a ring, box by box through the page
// table), warps 1 and 2 issue tcgen05.mma, one for each row tile, and clear V of keys that nobody sees (0 x NaN), warp 3
// works the pieces of the share out ahead, eight warps do the softmax, a thread per row: S from TMEM, maximum, exponentials, P
// back to TMEM over S as the A operand of O += P V.  A row tile's S is two key tiles ahead of its P (two buffers; with tiles of
// 128 keys and one buffer the tensor core waited: 8192 tokens causal 1547 us, so 632).  O stays in TMEM and is rescaled only
// when a row's maximum has grown by more than GROWTH octaves since the value its weights refer to, which is rare after the first
// tiles.  bf16 weights bear that like fp32 sums; fp16 weights begin at 2^(15 - GROWTH), so that the largest of its range is
// never passed and the small ones lose nothing above 2^-(29 - GROWTH) of the largest.
//
// The CTAs are persistent, one per SM, and share the work as in softmax_attention.cu: equal, contiguous pieces of all
// (block, key head) items laid end to end, in units of a key tile (of two where a block has one row tile).
//
// 16384 tokens causal, 32 heads over 8 of 128, bf16: 1.8 ms, 1.2 PFLOP/s, three quarters of a large matrix product's rate; 8192: 0.5
// ms (fp16: 2.0 and 0.57).  What is left: the two row tiles fall into step, and a block costs 4 us to finish and begin, which short
// histories (1000 keys, 17 tiles) feel as a third of their time.
#include "softmax_attention.cuh"

namespace {

using namespace rb_attn;

constexpr int KT = 64;                  // keys per tile
constexpr int MT = 128;                 // rows per row tile
// An item costs as much as FIXED units before its first key tile (measured: 4.4 us to finish one block and begin the next, 1.1
// us a unit): without them the shares with many short items would run half as long again as the others.
constexpr int FIXED = 4;
constexpr int THREADS = 384;            // 4 service warps, 2 x 4 softmax warps
template <bool BF16> constexpr float GROWTH = BF16 ? 8.f : 4.f;
// A row whose largest score (log2) is beyond this, on either side of 0, is reported: fp32 has no digit behind the point left there, and
// further out the fused operation that makes the exponents, whose product is not rounded as the maximum's was, loses the largest
// weight itself.  (Out to any size: the difference first, then its product, in a loop of its own: 2 to 3 % of a prompt's time.)
constexpr float FAR = 8388608.f;        // 2^23
constexpr uint32_t WAIT = 1u << 24;     // tries of a wait: some tenths of a second

template <int D> struct Cfg {
  static constexpr int CH = D / 64;
  static constexpr int TILE = KT * D * 2, Q_TILE = MT * D * 2;  // bytes of a K or V tile, of a Q tile
  static constexpr int STAGES = D == 64 ? 8 : 5;                // a K and a V tile each
  static constexpr int TAIL = 3 * 1024;              // shared memory is full to the last byte for D = 128
  static constexpr int SMEM = 2 * Q_TILE + STAGES * 2 * TILE + TAIL;
};

// One block of query tokens of a sequence: [t_lo, t_lo + tokens)
struct Block {
  int t_lo, tokens, two;                // two: a row tile each for the first and the rest of the tokens
  Span span;
  int units;                            // FIXED for the block itself, then one or two key tiles each
};

__device__ __forceinline__ int blocks_of(const Seq& s, int tpt) { return (s.len_q + 2 * tpt - 1) / (2 * tpt); }

__device__ __forceinline__ Block block_of(const Batch& p, const Seq& s, int i, int tpt) {
  Block b;
  b.t_lo = i * 2 * tpt;
  b.tokens = min(s.len_q - b.t_lo, 2 * tpt);
  b.two = b.tokens > tpt;
  b.span = span_of<KT>(p, s, b.t_lo, b.t_lo + b.tokens - 1);
  b.units = max(b.two ? b.span.tiles : (b.span.tiles + 1) / 2, 1) + FIXED;
  return b;
}

// The pieces of this CTA's share, one after another; every role walks its own copy.
struct Walk {
  int seq, block;
  long long base, pos, p0, p1;          // base: begin of the block's items (Hkv of them)
  // the current piece
  Seq s;
  Block b;
  int h, u0, u1;
  __device__ __forceinline__ bool next(const Batch& p, int tpt) {
    while (pos < p1 && seq < p.a.B + p.b.B) {
      s = seq_of(p, seq);
      const int n = blocks_of(s, tpt);
      if (block >= n) { ++seq; block = 0; continue; }
      b = block_of(p, s, block, tpt);
      const long long all = static_cast<long long>(b.units) * p.Hkv;
      if (pos >= base + all) { base += all; ++block; continue; }
      const uint32_t at = static_cast<uint32_t>(pos - base);                  // below units * Hkv: both are small numbers
      h = static_cast<int>(at / b.units);
      u0 = static_cast<int>(at - h * b.units);
      u1 = static_cast<int>(min(static_cast<long long>(b.units), u0 + (p1 - pos)));
      if (u1 <= FIXED) { done(); continue; }                                  // the next share begins the item
      return true;
    }
    return false;
  }
  __device__ __forceinline__ void done() { pos += u1 - u0; }
  // virtual key tiles of the piece
  __device__ __forceinline__ int v0() const { const int u = max(u0 - FIXED, 0); return b.two ? u : 2 * u; }
  __device__ __forceinline__ int v1() const { return min((b.two ? 1 : 2) * (u1 - FIXED), b.span.tiles); }
};

// A piece of the share as the roles need it; one thread works ahead and leaves it in shared memory.  Its key tiles are
// m = 0 .. n - 1 (tile v0 + m of the span).  Step e of the piece brings K of tile e and V of tile e - ahead through one slot
// of the ring (n + ahead steps): every row tile's S is computed two tiles ahead of its P.
struct Piece {
  Seq s;
  Span span;
  int n;                                // -1: there are no more pieces
  int v0, two, h, t_lo, tokens;
  int sink_end[2], first[2], end[2];    // row tile x sees the tiles m < sink_end[x] and first[x] <= m < end[x]
  int tiles[2];                         // how many of the piece's that are
  int clean_sinks, clean_lo, clean_hi;  // key tiles (by number) that some row sees to the last key
  int full_sinks, full_lo, full_hi;     // key tiles that every row sees to the last key
  int whole;                            // the piece is the whole item
  int cut;                              // else: where its results go
};

struct Bars {
  uint64_t full[8], empty[8];           // ring
  uint64_t q_full, q_empty, fixed, drain[2], swap[2];
  uint64_t s_full[2][2], p_full[2][2];  // of row tile x, buffer b
  uint64_t o_done[2];                   // every product with V
  uint64_t o_full[2], o_empty[2];       // the piece's result is there, has been read
  uint64_t piece_full[2], piece_empty[2];
};
static_assert(sizeof(Bars) <= 512 && sizeof(Piece) <= 216, "the tail's layout");
constexpr int READERS = 1 + 2 + 8;      // warps that read a piece: loads, tensor core, softmax

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// one lane of a converged warp, which the compiler takes as issuing for it (a test of the lane's number made a loop of it)
__device__ __forceinline__ bool elect() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}
// (address 32-byte aligned)
__device__ __forceinline__ void store32(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// rb::mbar_wait without the sleep between tries: the waits here are on the critical path and short
__device__ __forceinline__ bool spin_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
  for (uint32_t it = 0; it < WAIT; ++it) {
    if (rb::mbar_try_wait(bar, parity)) return true;
    if ((it & 1023) == 1023 && *abort_flag) return false;
  }
  *abort_flag = 1;
  if (status) atomicCAS(status, 0, RB_ERR_MBAR_TIMEOUT);
  return false;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
attn_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const Batch p, const Outs w) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];                           // the swizzle wants it; nothing is left to align by hand
  uint8_t* q_s = smem;                                                        // [2][Q_TILE]
  uint8_t* ring = smem + 2 * C::Q_TILE;                                       // [STAGES][K, V][TILE]
  uint8_t* tail = ring + C::STAGES * 2 * C::TILE;
  Bars* bars = reinterpret_cast<Bars*>(tail);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 516);
  int* found = reinterpret_cast<int*>(tail + 520);                            // sequence, block
  long long* found_base = reinterpret_cast<long long*>(tail + 528);
  long long* wsum = reinterpret_cast<long long*>(ring + 4 * THREADS);         // [12], before the first load like first_item
  int* wcnt = reinterpret_cast<int*>(ring + 4 * THREADS + 128);               // [12]
  float* ml = reinterpret_cast<float*>(tail + 592);                           // [2][MT][2]
  Piece* pieces = reinterpret_cast<Piece*>(tail + 2640);                      // [2]
  int* first_item = reinterpret_cast<int*>(ring);                             // [THREADS], before the first load
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tpt = MT / p.G;                                                   // tokens per row tile
  const int nb = p.a.B + p.b.B;

  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) { rb::mbar_init(&bars->full[i], 1); rb::mbar_init(&bars->empty[i], 2); }
    rb::mbar_init(&bars->q_full, 1); rb::mbar_init(&bars->q_empty, 2);
    rb::mbar_init(&bars->fixed, 2);
    for (int i = 0; i < 2; ++i) {
      for (int j = 0; j < 2; ++j) { rb::mbar_init(&bars->s_full[i][j], 1); rb::mbar_init(&bars->p_full[i][j], MT / 32); }
      rb::mbar_init(&bars->o_done[i], 1); rb::mbar_init(&bars->o_full[i], 1); rb::mbar_init(&bars->o_empty[i], MT / 32);
      rb::mbar_init(&bars->swap[i], 2 * MT / 32); rb::mbar_init(&bars->drain[i], 1);
      rb::mbar_init(&bars->piece_full[i], 1); rb::mbar_init(&bars->piece_empty[i], READERS);
    }
    *abort_flag = 0;
    rb::mbar_fence_init();
  }
  if (warp == 2) { rb::tmem_alloc(tmem_slot, 512); rb::tmem_relinquish(); }
  launch_dependents();

  // ---- this CTA's share.  Blocks per sequence differ, so they are counted first and then dealt to the threads evenly.
  const int per = (nb + THREADS - 1) / THREADS;
  int n_mine = 0;
  for (int i = tid * per; i < min((tid + 1) * per, nb); ++i) n_mine += blocks_of(seq_of(p, i), tpt);
  int seq0 = tid * per, blk0 = 0, n_own = n_mine;                             // this thread's blocks: from (seq0, blk0) on
  if (__syncthreads_or(n_mine > 8)) {
    // some threads have many: deal them all out anew
    int n_incl = n_mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, n_incl, o);
      if (lane >= o) n_incl += x;
    }
    if (lane == 31) wcnt[warp] = n_incl;
    __syncthreads();
    int n_all = 0, n_before = n_incl - n_mine;
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) n_before += wcnt[i];
      n_all += wcnt[i];
    }
    first_item[tid] = n_before;
    __syncthreads();
    const int ipt = (n_all + THREADS - 1) / THREADS;
    const int my_first = tid * ipt;
    n_own = max(min(my_first + ipt, n_all) - my_first, 0);
    if (n_own > 0) {
      // the last thread whose first block is not after this one's owns it
      int lo = 0, hi = THREADS - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_item[mid] <= my_first) lo = mid; else hi = mid - 1;
      }
      int left = my_first - first_item[lo];
      seq0 = lo * per;
      for (;;) {
        const int n = blocks_of(seq_of(p, seq0), tpt);
        if (left < n) { blk0 = left; break; }
        left -= n;
        ++seq0;
      }
    }
  }
  auto each = [&](auto&& f) {                                                 // f(seq, block, units of all its items)
    int sq = seq0, bl = blk0;
    for (int i = 0; i < n_own; ++i) {
      Seq s = seq_of(p, sq);
      while (bl >= blocks_of(s, tpt)) { ++sq; bl = 0; s = seq_of(p, sq); }
      if (f(sq, bl, static_cast<long long>(block_of(p, s, bl, tpt).units) * p.Hkv)) return;
      ++bl;
    }
  };
  long long mine = 0;
  each([&](int, int, long long n) { mine += n; return false; });
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  long long total = 0, before = incl - mine;
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) before += wsum[i];
    total += wsum[i];
  }
  const int cta = blockIdx.x;
  const Shares sh(total, gridDim.x);
  Walk walk;
  walk.p0 = cta < sh.n ? sh.begin(cta) : 0;
  walk.p1 = cta < sh.n ? sh.begin(cta + 1) : 0;
  if (walk.p0 < walk.p1 && before <= walk.p0 && walk.p0 < before + mine) {
    long long base = before;
    each([&](int sq, int bl, long long n) {
      if (walk.p0 < base + n) { found[0] = sq; found[1] = bl; *found_base = base; return true; }
      base += n;
      return false;
    });
  }
  rb::fence_proxy_async_smem();                                               // first_item's words are the ring's now
  rb::tc_fence_before();
  __syncthreads();
  rb::tc_fence_after();
  const uint32_t tmem = *tmem_slot;                                           // S / P of row tile w at w * 128, O at 256 + w * 128
  bool gave_up = false;
  int n_piece = 0;
  // A warp gives up as one, and arrives as one by lane 0 (arrivals on one word are served one after another).
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const int ok = !gave_up && spin_wait(bar, parity, abort_flag, p.status);
    if (!__all_sync(0xffffffffu, ok)) gave_up = true;
    return !gave_up;
  };
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) rb::mbar_arrive(bar);
  };
  // the next piece, or null when there are no more (or a wait ran out); a warp gives up as one
  auto next_piece = [&]() -> const Piece* {
    if (!wait(&bars->piece_full[n_piece & 1], (n_piece >> 1) & 1)) return nullptr;
    const Piece* q = pieces + (n_piece & 1);
    return q->n < 0 ? nullptr : q;
  };
  auto done_piece = [&]() { arrive(&bars->piece_empty[n_piece & 1]); ++n_piece; };

  if (warp == 3) {
    // ------------------------------------------------------------------ pieces
    if (lane == 0) {
      walk.seq = found[0]; walk.block = found[1]; walk.base = *found_base; walk.pos = walk.p0;
      if (walk.p0 >= walk.p1) walk.pos = walk.p1 = 0;
      Meta mt;
      mt.valid = 0;
      for (;; ++n_piece) {
        const bool more = walk.next(p, tpt);
        if (!spin_wait(&bars->piece_empty[n_piece & 1], ((n_piece >> 1) & 1) ^ 1, abort_flag, p.status)) break;
        Piece& q = pieces[n_piece & 1];
        q.n = -1;
        if (more) {
          const Block& b = walk.b;
          q.s = walk.s; q.span = b.span; q.v0 = walk.v0(); q.n = max(walk.v1() - walk.v0(), 0); q.two = b.two; q.h = walk.h;
          q.t_lo = b.t_lo; q.tokens = b.tokens;
          const int skip = b.span.first - b.span.sink_tiles + q.v0;            // tile number - m, past the sinks
          for (int x = 0; x < 2; ++x) {
            const int lo = b.t_lo + x * tpt;
            const Span sx = span_of<KT>(p, walk.s, lo, min(lo + tpt, b.t_lo + b.tokens) - 1);
            q.sink_end[x] = (sx.sinks + KT - 1) / KT - q.v0;               // (past sink_tiles nothing is skipped)
            q.first[x] = sx.first - skip;
            q.end[x] = sx.end - skip;
            // sinks first, then the range, without what both count
            const int se = min(max(q.sink_end[x], 0), q.n), fi = min(max(q.first[x], se), q.n), en = min(max(q.end[x], fi), q.n);
            q.tiles[x] = b.two ? se + en - fi : (q.n + 1 - x) / 2;
          }
          const bool win = walk.s.causal && p.window > 0;
          q.clean_sinks = b.span.sinks / KT; q.clean_lo = (b.span.lo + KT - 1) / KT; q.clean_hi = b.span.hi / KT;
          const int upto = max(walk.s.causal ? b.span.p_min + 1 : b.span.hi, 0);
          q.full_sinks = win ? min(p.sinks, upto) / KT : 0;
          q.full_lo = win ? (max(b.span.p_max - p.window + 1, 0) + KT - 1) / KT : 0;
          q.full_hi = upto / KT;
          q.whole = walk.u0 <= FIXED && walk.u1 == b.units;
          q.cut = cta * 2 + (walk.pos == walk.p0 ? 0 : 1);
          const long long t0 = walk.pos - walk.u0;
          if (walk.pos == walk.p0 && walk.u0 > FIXED && sh.begin(cta - 1) <= t0 + FIXED) {
            // the first border between this item's tiles: another kernel joins its pieces
            mt.valid = 1; mt.seq = walk.seq; mt.row0 = b.t_lo * p.G; mt.rows = b.tokens * p.G; mt.h = walk.h;
            mt.c0 = cta - 1;
            mt.c1 = sh.of(t0 + b.units - 1);
            mt.first = 2 * mt.c0 + (sh.begin(mt.c0) >= t0 ? 0 : 1);           // its share's first piece or its last
          }
          walk.done();
        }
        rb::mbar_arrive(&bars->piece_full[n_piece & 1]);
        if (!more) break;
      }
      w.meta[cta] = mt;
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------------ loads: a lane per box of K, a lane per box of V
    int st = 0, n_q = 0, last = 0;
    uint32_t par = 1;                                                         // of `empty`
    const int boxes = KT / p.box_rows;
    const int my_kind = lane / (boxes * C::CH);                               // 0: K, 1: V
    const int my_box = lane / C::CH % boxes, my_chunk = lane % C::CH;
    while (const Piece* q = next_piece()) {
      const bool two = q->two;
      const int v0 = q->v0, n = q->n, col = q->h * D + my_chunk * 64, q_head = q->h * p.G;
      const Seq s = q->s;
      const Span sp = q->span;
      const int q_row = s.q_begin + q->t_lo;
      done_piece();
      if (n == 0) continue;
      // Rows of the boxes, looked up for 32 / boxes tiles at a time (a division, a page id: slow one by one): lane l holds
      // box l % boxes of tile l / boxes of a batch; V lags K by less than a batch.
      const int batch = 32 / boxes;
      int rows_now = 0, rows_before = 0, begin = 0;                           // begin: first tile of rows_now
      auto look_up = [&](int m0) {
        const int m = m0 + lane / boxes, v = v0 + m;
        const int k0 = (v < sp.sink_tiles ? v : sp.first + v - sp.sink_tiles) * KT;
        rows_before = rows_now;
        rows_now = m < n && lane < batch * boxes ? box_row(p, s, sp, k0 + (lane % boxes) * p.box_rows) : p.total_rows;
        begin = m0;
      };
      look_up(0);
      if (!wait(&bars->q_empty, (n_q & 1) ^ 1)) break;
      ++n_q;
      if (lane == 0) {
        rb::mbar_expect_tx(&bars->q_full, (two ? 2 : 1) * C::CH * p.G * tpt * 128);
        for (int t = 0; t < (two ? 2 : 1); ++t)
#pragma unroll
          for (int c = 0; c < C::CH; ++c)
            rb::tma_load_3d(q_s + t * C::Q_TILE + c * (MT * 128), &tm_q, &bars->q_full, c * 64, q_head, q_row + t * tpt);
      }
      const int ahead = two ? 2 : 4;
      for (int e = 0; e < n + ahead; ++e) {
        if (e == begin + batch) look_up(e);
        const int m = my_kind ? e - ahead : e;                                // this lane's tile
        const int src = (m - begin) * boxes + my_box;
        const int now = __shfl_sync(0xffffffffu, rows_now, src & 31), old = __shfl_sync(0xffffffffu, rows_before, (src + batch * boxes) & 31);
        const int row = (m >= begin ? now : old) + my_kind * p.page_size;
        if (!wait(&bars->empty[st], par)) break;
        if (lane == 0) rb::mbar_expect_tx(&bars->full[st], ((e < n ? 1 : 0) + (e >= ahead ? 1 : 0)) * C::TILE);
        __syncwarp();
        if (my_kind < 2 && m >= 0 && m < n)
          rb::tma_load_2d(ring + (st * 2 + my_kind) * C::TILE + my_chunk * (KT * 128) + my_box * p.box_rows * 128, &tm_kv, &bars->full[st], col, row);
        ++last;
        if (++st == C::STAGES) { st = 0; par ^= 1; }
      }
    }
    if (gave_up && lane == 0)                                                 // copies in flight end before the kernel does
      for (int i = max(last - C::STAGES, 0); i < last; ++i)
        for (int k = 0; k < (1 << 16) && !rb::mbar_try_wait(&bars->full[i % C::STAGES], (i / C::STAGES) & 1); ++k) {}
  } else if (warp < 3) {
    // ------------------------------------------------------------------ tensor core: warp 1 + x for row tile x
    // Each of the two walks the whole ring and gives every tile back, used or not, so both keep its order.
    const int x = warp - 1;
    const uint32_t idesc_s = rb::umma_idesc(MT, KT, 0, 0, BF16), idesc_o = rb::umma_idesc(MT, D, 0, 1, BF16);
    const uint32_t t_s = tmem + x * 128, t_o = tmem + 256 + x * 128;          // S and P: two buffers of KT columns
    // descriptors of a tile at offset 0; an address is added to the low word in units of 16 bytes
    const uint32_t ring_at = rb::smem_u32(ring) >> 4;
    const uint64_t d_k = rb::umma_smem_desc(0, 16, 1024) + ring_at, d_v = rb::umma_smem_desc(0, KT * 128, 1024) + ring_at + (C::TILE >> 4);
    const uint64_t d_q = rb::umma_smem_desc(0, 16, 1024) + (rb::smem_u32(q_s) >> 4);
    int st = 0;
    uint32_t par = 0, par_q = 0, par_o = 1, par_fix = 0, n_s = 0, n_p = 0;   // n_s, n_p: this row tile's S and P so far
    // the ring's slot goes back once what was issued so far is done
    auto pass = [&](bool used) {
      if (elect()) {
        if (used) rb::umma_commit(&bars->empty[st]); else rb::mbar_arrive(&bars->empty[st]);
      }
      if (++st == C::STAGES) { st = 0; par ^= 1; }
    };
    auto mma_s = [&](int q_tile) {                                            // S = Q K^T with the slot's K
      rb::tc_fence_after();
      const uint32_t buf = n_s++ & 1;
      if (elect()) {
        const uint64_t dq = d_q + static_cast<uint32_t>(q_tile * (C::Q_TILE >> 4)), dk = d_k + static_cast<uint32_t>(st * (C::TILE >> 3));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          rb::umma_f16_ss(t_s + buf * KT, dq + (((kk / 4) * (MT * 128) + (kk % 4) * 32) >> 4),
                          dk + (((kk / 4) * (KT * 128) + (kk % 4) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
        rb::umma_commit(&bars->s_full[x][buf]);
      }
    };
    while (const Piece* q = next_piece()) {
      const bool two = q->two;
      int left = q->tiles[x];                                                 // of this row tile's products with V
      const int n = q->n;
      const int v0 = q->v0, sink_tiles = q->span.sink_tiles, skip = q->span.first - sink_tiles;
      const int c_sinks = q->clean_sinks, c_lo = q->clean_lo, c_hi = q->clean_hi;
      const int hi = q->span.hi, lo = q->span.lo, sinks = q->span.sinks;
      const int se = q->sink_end[x], fi = q->first[x], en = q->end[x];
      done_piece();
      if (n == 0) continue;
      bool started = false;
      auto mine = [&](int m) { return two ? m < se || (m >= fi && m < en) : (m & 1) == x; };
      if (!wait(&bars->q_full, par_q)) break;
      par_q ^= 1;
      const int ahead = two ? 2 : 4;
      // steps whose V is this row tile's and needs no clearing
      const int clean0 = max(c_lo - skip, sink_tiles) - v0, clean1 = c_hi - skip - v0;
      const int plain0 = max(clean0, two ? fi : 0) + ahead, plain1 = min(clean1, two ? min(en, n) : n) + ahead;
      const uint32_t q_at = (two ? x : 0) * (C::Q_TILE >> 4);
      for (int e = 0; e < n + ahead; ++e) {
        const int m = e - ahead;
        if (!two && (e & 1) != x) {                                           // the other warp's step
          if (!wait(&bars->full[st], par)) break;
          if (e == n - 1 && elect()) rb::umma_commit(&bars->q_empty);
          pass(false);
          continue;
        }
        if (e >= plain0 && e < plain1 && started) {
          // the same as below, without its questions: this is where the time goes
          const bool use_k = e < n && mine(e);
          if (!wait(&bars->full[st], par)) break;
          const uint32_t bp = n_p & 1, bs = n_s & 1;
          if (!wait(&bars->p_full[x][bp], (n_p >> 1) & 1)) break;
          ++n_p;
          n_s += use_k;
          rb::tc_fence_after();
          if (elect()) {
            const uint32_t at = st * (C::TILE >> 3);
            const uint64_t dv = d_v + at, dq = d_q + q_at, dk = d_k + at;
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk) rb::umma_f16_ts(t_o, t_s + bp * KT + kk * 8, dv + kk * 128, idesc_o, 1u);
            rb::umma_commit(&bars->o_done[x]);
            if (left == 1) rb::umma_commit(&bars->o_full[x]);
            if (use_k) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                rb::umma_f16_ss(t_s + bs * KT, dq + (((kk / 4) * (MT * 128) + (kk % 4) * 32) >> 4),
                                dk + (((kk / 4) * (KT * 128) + (kk % 4) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
              rb::umma_commit(&bars->s_full[x][bs]);
            }
            rb::umma_commit(&bars->empty[st]);
            if (e == n - 1) rb::umma_commit(&bars->q_empty);
          }
          --left;
          if (++st == C::STAGES) { st = 0; par ^= 1; }
          continue;
        }
        const bool use_k = e < n && mine(e), use_v = m >= 0 && mine(m);
        if (!wait(&bars->full[st], par)) break;
        if (m >= 0 && (two || use_v)) {
          // V of keys that no row of the block sees may be anything: clear it
          const int v = v0 + m, t = v < sink_tiles ? v : v + skip;
          if (!(t < c_sinks || (t >= c_lo && t < c_hi))) {
            uint8_t* tile = ring + (st * 2 + 1) * C::TILE;
            for (int i = two ? lane * 2 + x : lane; i < KT; i += two ? 64 : 32) {
              const int j = t * KT + i;
              if (j < hi && (j >= lo || j < sinks)) continue;
              uint4* row = reinterpret_cast<uint4*>(tile + i * 128);
#pragma unroll
              for (int c = 0; c < C::CH; ++c)
#pragma unroll
                for (int u = 0; u < 8; ++u) row[c * (KT * 8) + ((u + lane) & 7)] = make_uint4(0, 0, 0, 0);
            }
            rb::fence_proxy_async_smem();
            __syncwarp();
            if (two) {                                                        // the other half of the rows is the other warp's
              arrive(&bars->fixed);
              if (!wait(&bars->fixed, par_fix)) break;
              par_fix ^= 1;
            }
          }
        }
        if (use_v) {                                                          // O (+)= P V
          if (!started) {
            if (!wait(&bars->o_empty[x], par_o)) break;
            par_o ^= 1;
          }
          const uint32_t buf = n_p & 1;
          if (!wait(&bars->p_full[x][buf], (n_p >> 1) & 1)) break;
          ++n_p;
          rb::tc_fence_after();
          if (elect()) {
            const uint64_t dv = d_v + static_cast<uint32_t>(st * (C::TILE >> 3));
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk)
              rb::umma_f16_ts(t_o, t_s + buf * KT + kk * 8, dv + kk * 128, idesc_o, (kk > 0 || started) ? 1u : 0u);
            rb::umma_commit(&bars->o_done[x]);
            if (left == 1) rb::umma_commit(&bars->o_full[x]);
          }
          --left;
          started = true;
        }
        if (use_k) mma_s(two ? x : 0);
        pass(use_k || use_v);
        if (e == n - 1 && elect()) rb::umma_commit(&bars->q_empty);           // the last S is issued: Q may go
      }
      if (gave_up) break;
    }
    if (gave_up && lane == 0) {                                               // nothing of ours still runs when TMEM is freed
      rb::umma_commit(&bars->drain[x]);
      for (int k = 0; k < (1 << 16) && !rb::mbar_try_wait(&bars->drain[x], 0); ++k) {}
    }
  } else {
    // ------------------------------------------------------------------ softmax: thread = row
    const int x = (warp - 4) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_sel + x * 128, t_o = tmem + lane_sel + 256 + x * 128;
    const int my_tok = row / p.G, my_head = row % p.G;                         // of the row tile, of the group
    uint32_t n_s = 0, par_o = 0, par_swap = 0;                                  // key tiles so far; bit y: of row tile y's o_full
    while (const Piece* q = next_piece()) {
      const bool two = q->two;
      const int n = q->n;
      float m_ref = -INFINITY, sum = 0.f;                                      // log2 domain
      bool any = false;
      {
        const int v0 = q->v0, sink_tiles = q->span.sink_tiles, skip = q->span.first - sink_tiles;
        const int se = q->sink_end[x], fi = q->first[x], en = q->end[x];
        const int full_s = q->full_sinks, full_lo = q->full_lo, full_hi = q->full_hi;
        const int pos = q->t_lo + (two ? x * tpt : 0) + my_tok + q->s.delta();
        for (int m = two ? 0 : x; m < n; m += two ? 1 : 2) {
          if (two && !(m < se || (m >= fi && m < en))) continue;
          const int t = v0 + m < sink_tiles ? v0 + m : v0 + m + skip;
          const uint32_t buf = n_s & 1;
          if (!wait(&bars->s_full[x][buf], (n_s >> 1) & 1)) break;
          rb::tc_fence_after();
          uint32_t sr[KT / 32][32];
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) rb::tmem_ld_32x32(t_s + buf * KT + c * 32, sr[c]);
          rb::tmem_ld_wait();
          if (!(t < full_s || (t >= full_lo && t < full_hi))) {
#pragma unroll
            for (int c = 0; c < KT / 32; ++c) {
              const uint32_t seen = seen_keys(pos, t * KT + c * 32, q->s.len_k, q->s.causal, p.window, p.sinks);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen & (1u << e))) sr[c][e] = 0xff800000u;
            }
          }
          float mx[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t* v = &sr[c >> 1][(c & 1) * 16];
            mx[c] = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[15]));
#pragma unroll
            for (int e = 1; e < 15; e += 2) mx[c] = fmaxf(mx[c], fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
          }
          const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;   // scale > 0 in this kernel
          // O and the sum refer to m_ref; only a row whose weights would pass 2^TOP (or its first weight) moves it
          constexpr float START = BF16 ? 0.f : WeightTop<BF16> - GROWTH<BF16>, TOP = START + GROWTH<BF16>;
          const bool grow = m_new > (BF16 ? m_ref + TOP : __fadd_rd(m_ref, TOP)) || (m_ref == -INFINITY && m_new > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float m_next = BF16 ? m_new : __fsub_ru(m_new, START);
            const float f = grow ? (m_ref == -INFINITY ? 0.f : exp2_approx(m_ref - m_next)) : 1.f;
            if (grow) m_ref = m_next;
            sum *= f;
            if (any) {
              // once the product with the tile before is done, O is at rest until this tile's P is there
              if (!wait(&bars->o_done[x], (n_s - 1) & 1)) break;
              rb::tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                rb::tmem_ld_32x16(t_o + c * 16, o);
                rb::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                rb::tmem_st_32x16(t_o + c * 16, o);
              }
              rb::tmem_st_wait();
            }
          }
          const float base = m_ref == -INFINITY ? 0.f : m_ref;
          const float2 sc = make_float2(p.scale_log2, p.scale_log2), nb2 = make_float2(-base, -base);
          float2 acc0 = make_float2(sum, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float2 a = fma2(make_float2(__uint_as_float(sr[c][e]), __uint_as_float(sr[c][e + 1])), sc, nb2);
              float2 b = fma2(make_float2(__uint_as_float(sr[c][e + 2]), __uint_as_float(sr[c][e + 3])), sc, nb2);
              a.x = exp2_approx(a.x); a.y = exp2_approx(a.y); b.x = exp2_approx(b.x); b.y = exp2_approx(b.y);
              acc0 = add2(acc0, a);
              acc1 = add2(acc1, b);
              pk[e >> 1] = pack16<BF16>(a.x, a.y);
              pk[(e >> 1) + 1] = pack16<BF16>(b.x, b.y);
            }
            rb::tmem_st_32x16(t_s + buf * KT + c * 16, pk);
          }
          sum = (acc0.x + acc0.y) + (acc1.x + acc1.y);
          rb::tmem_st_wait();
          rb::tc_fence_before();
          arrive(&bars->p_full[x][buf]);
          ++n_s;
          any = true;
        }
      }
      // ---- the piece's result: columns [c_lo, c_hi) of the row are this thread's to write
      int c_lo = 0, c_hi = D;
      float f0 = x == 0 ? 1.f : 0.f, f1 = 1.f - f0, l = sum, m_all = m_ref;
      const bool mine = q->tiles[x] > 0;
      const uint32_t had = (q->tiles[0] > 0 ? 1u : 0u) | (q->tiles[1] > 0 ? 2u : 0u);
      if (fabsf(m_ref) >= FAR && fabsf(m_ref) < INFINITY && my_tok < min(q->tokens - (two ? x * tpt : 0), tpt) && p.status)
        atomicCAS(p.status, 0, RB_ERR_RANGE);
      if (!two) {
        ml[(x * MT + row) * 2] = m_ref; ml[(x * MT + row) * 2 + 1] = sum;
        arrive(&bars->swap[0]);
        wait(&bars->swap[0], par_swap);
        const float m0 = ml[row * 2], l0 = ml[row * 2 + 1], m1 = ml[(MT + row) * 2], l1 = ml[(MT + row) * 2 + 1];
        m_all = fmaxf(m0, m1);
        const float bm = m_all == -INFINITY ? 0.f : m_all;
        f0 = exp2_approx(m0 - bm); f1 = exp2_approx(m1 - bm);
        l = f0 * l0 + f1 * l1;
        c_lo = x * (D / 2); c_hi = c_lo + D / 2;
      }
      const bool read0 = two ? x == 0 && mine : q->tiles[0] > 0, read1 = two ? x == 1 && mine : q->tiles[1] > 0;
      if (read0) wait(&bars->o_full[0], par_o & 1);
      if (read1) wait(&bars->o_full[1], par_o >> 1);
      par_o ^= had;
      rb::tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float lse2 = l == 0.f ? -INFINITY : m_all + log2f(l);
      f0 *= inv; f1 *= inv;
      if (!gave_up) {
        const int r_cut = two ? x * tpt * p.G + row : row;                      // row of the block
        const int tok = (two ? x * tpt : 0) + my_tok;
        const bool live = row < tpt * p.G && tok < q->tokens;
        // where row_out would send it, without its divisions
        const int t = q->s.q_begin + q->t_lo + tok, head = q->h * p.G + my_head;
        uint16_t* dst16 = nullptr;
        float *dst32 = nullptr, *dst_lse;
        float lse = lse2;
        if (!q->whole) {
          const int cut = q->cut * TILE_ROWS + r_cut;
          dst32 = w.cut_o + static_cast<long long>(cut) * D;
          dst_lse = w.cut_lse + cut;
        } else if (w.part_o) {
          const long long at = (static_cast<long long>(q->s.part) * p.Tq + t) * p.H + head;
          dst32 = w.part_o + at * D;
          dst_lse = w.part_lse + at;
        } else {
          dst16 = reinterpret_cast<uint16_t*>(w.out) + t * w.ld_o + head * D;
          dst_lse = w.lse ? w.lse + (static_cast<long long>(t) * p.H + head) : nullptr;
          lse = lse2 * LN2;
        }
        if (live && c_lo == 0 && dst_lse) *dst_lse = lse;
#pragma unroll 1
        for (int c = c_lo; c < c_hi; c += 32) {
          uint32_t a[32];
          float o[32];
          if (read0) {
            rb::tmem_ld_32x32(tmem + lane_sel + 256 + c, a);
            rb::tmem_ld_wait();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = read0 ? f0 * __uint_as_float(a[e]) : 0.f;
          if (read1) {
            rb::tmem_ld_32x32(tmem + lane_sel + 384 + c, a);
            rb::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(f1, __uint_as_float(a[e]), o[e]);
          }
          // 32 bytes a store: a row per thread means a line per lane, and what counts is how many stores there are
          if (live && dst16) {
#pragma unroll
            for (int e = 0; e < 32; e += 16) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = pack16<BF16>(o[e + 2 * i], o[e + 2 * i + 1]);
              store32(dst16 + c + e, v);
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t v[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(o[e + i]);
              store32(dst32 + c + e, v);
            }
          }
        }
      }
      rb::tc_fence_before();
      if (!two) {                                                               // both sets of warps read both results
        arrive(&bars->swap[1]);
        wait(&bars->swap[1], par_swap);
        par_swap ^= 1;
      }
      if (mine) arrive(&bars->o_empty[x]);
      done_piece();
    }
  }
  __syncwarp();
  rb::tc_fence_before();
  __syncthreads();
  if (warp == 2) rb::tmem_dealloc(tmem, 512);
  if (tid == 0) wait_before();                                                // what ran before is done when this kernel is
}

// q as [Tq][H][D]: boxes of 64 elements x G heads x the tokens of a row tile
int make_map_q(CUtensorMap* map, const Batch& p, int D, int tpt, bool is_bf16) {
  rb_host::EncodeTiledFn fn = rb_host::encode_tiled_fn();
  if (!fn) return -1;
  rb_host::bind_context(p.q);
  cuuint64_t dim[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(p.H), static_cast<cuuint64_t>(p.Tq)};
  cuuint64_t stride[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(p.ld_q) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.G), static_cast<cuuint32_t>(tpt)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p.q), dim,
                        stride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -(1000 + static_cast<int>(r));
}

template <int D, bool BF16>
int launch(const Batch& p, const Outs& w, const void* cache, int n_cta, bool after, cudaStream_t st) {
  CUtensorMap tq, tkv;
  int rc = make_map_q(&tq, p, D, MT / p.G, BF16);
  if (rc) return rc;
  rc = rb_host::make_map_2d(&tkv, cache, p.total_rows, static_cast<long long>(p.Hkv) * D, static_cast<long long>(p.Hkv) * D, 64, p.box_rows, BF16);
  if (rc) return rc;
  static std::atomic<unsigned long long> done{0};
  rc = rb_host::allow_smem(attn_tiles_kernel<D, BF16>, Cfg<D>::SMEM, done);
  if (rc) return rc;
  return launch_kernel(after, attn_tiles_kernel<D, BF16>, dim3(n_cta), dim3(THREADS), Cfg<D>::SMEM, st, tq, tkv, p, w);
}

}  // namespace

int rb_attn::launch_tiles(const Batch& batch, const Outs& w, const void* cache, int D, bool is_bf16, int n_cta, bool after, cudaStream_t st) {
  Batch p = batch;
  p.box_rows = p.page_size % 64 == 0 ? 64 : p.page_size % 32 == 0 ? 32 : 16;
  if (D == 64) return is_bf16 ? launch<64, true>(p, w, cache, n_cta, after, st) : launch<64, false>(p, w, cache, n_cta, after, st);
  return is_bf16 ? launch<128, true>(p, w, cache, n_cta, after, st) : launch<128, false>(p, w, cache, n_cta, after, st);
}
