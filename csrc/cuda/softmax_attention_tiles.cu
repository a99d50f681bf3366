// Softmax attention over the paged KV cache for many query rows per sequence (prompts, new tokens over a long history, a
// group of requests behind a common prefix), forward, on tcgen05 / TMEM (sm_100a).  The mathematics is that of
// softmax_attention.cu: one pass over K and V with a running maximum and sum in fp32.
//
// Bound: the matrix rate and, equally, the exponentials: a 128 x 128 block costs 2 x 128 x 128 x D multiply-adds (1024
// cycles of the tensor core for D = 128) and 16384 exponentials (1024 cycles of the special function units).  So two
// blocks are always in flight, one in the tensor core while the other is in the softmax warps:
//   * 256 rows (two row tiles of 128: 128 / G tokens x the G query heads that share a key head) walk the same key tiles, or
//   * where a block has 128 rows or fewer, one row tile takes even key tiles with one set of warps and odd ones with
//     the other; the two results are joined from TMEM at the end.
// Roles: one thread issues TMA loads (Q once per block, then K and V tiles of 128 keys through a ring, box by box through the page
// table), one issues tcgen05.mma, one warp clears V of keys that nobody sees (0 x NaN), eight warps do the softmax, a
// thread per row: S from TMEM, maximum, exponentials, P back to TMEM over S as the A operand of O += P V.  O stays in TMEM
// and is rescaled only when a row's maximum has grown by more than 2^8 since the value its weights refer to, which fp32
// sums and 16-bit weights (a floating-point type: no precision lost) bear and which is rare after the first tiles.
//
// The CTAs are persistent, one per SM, and share the work as in softmax_attention.cu: equal, contiguous pieces of all
// (block, key head) items laid end to end, in units of two 128 x 128 blocks.
#include "softmax_attention.cuh"

namespace {

using namespace rb_attn;

constexpr int KT = 128;                 // keys per tile
constexpr int MT = 128;                 // rows per row tile
constexpr int THREADS = 384;            // 4 service warps, 2 x 4 softmax warps
constexpr int WAIT = 1 << 22;

template <int D> struct Cfg {
  static constexpr int CH = D / 64;
  static constexpr int TILE = KT * D * 2;                       // bytes of a Q, K or V tile
  static constexpr int STAGES = D == 64 ? 10 : 5;
  static constexpr int TAIL = 3072;               // shared memory is full to the last byte for D = 128
  static constexpr int SMEM = (2 + STAGES) * TILE + TAIL;
};

// One block of query tokens of a sequence: [t_lo, t_lo + tokens)
struct Block {
  int t_lo, tokens, two;                // two: a row tile each for the first and the rest of the tokens
  Span span;
  int units;
};

__device__ __forceinline__ int blocks_of(const Seq& s, int tpt) { return (s.len_q + 2 * tpt - 1) / (2 * tpt); }

__device__ __forceinline__ Block block_of(const Batch& p, const Seq& s, int i, int tpt) {
  Block b;
  b.t_lo = i * 2 * tpt;
  b.tokens = min(s.len_q - b.t_lo, 2 * tpt);
  b.two = b.tokens > tpt;
  b.span = span_of<KT>(p, s, b.t_lo, b.t_lo + b.tokens - 1);
  b.units = max(b.two ? b.span.tiles : (b.span.tiles + 1) / 2, 1);
  return b;
}

// The pieces of this CTA's share, one after another; every role walks its own copy.
struct Walk {
  int seq, block, n_sh;
  long long base, pos, p0, p1, total;   // base: begin of the block's items (Hkv of them)
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
      h = static_cast<int>((pos - base) / b.units);
      u0 = static_cast<int>((pos - base) % b.units);
      u1 = static_cast<int>(min(static_cast<long long>(b.units), u0 + (p1 - pos)));
      return true;
    }
    return false;
  }
  __device__ __forceinline__ void done() { pos += u1 - u0; }
  // virtual key tiles of the piece
  __device__ __forceinline__ int v0() const { return b.two ? u0 : 2 * u0; }
  __device__ __forceinline__ int v1() const { return min(b.two ? u1 : 2 * u1, b.span.tiles); }
};

// Where the tiles of a piece with n key tiles stand in the order of loads, which is the order of first use:
// K0 V0 K1 V1 ... when both row tiles use every key tile, K0 K1 V0 K2 V1 ... when they take turns.
__device__ __forceinline__ int k_index(bool two, int m) { return two ? 2 * m : m + max(m - 1, 0); }
__device__ __forceinline__ int v_index(bool two, int m, int n) { return two ? 2 * m + 1 : m + min(n, m + 2); }

// which key tiles row tile w of a block sees (the other's extra tiles at the ends are left out)
struct Active {
  int sink_end, first, end;
  __device__ __forceinline__ bool operator()(int tile) const { return tile < sink_end || (tile >= first && tile < end); }
};
__device__ __forceinline__ Active active_of(const Batch& p, const Seq& s, const Block& b, int w, int tpt) {
  Active a;
  const int lo = b.two ? b.t_lo + w * tpt : b.t_lo;
  const int hi = b.two ? min(lo + tpt, b.t_lo + b.tokens) - 1 : b.t_lo + b.tokens - 1;
  const Span sp = span_of<KT>(p, s, lo, hi);
  a.sink_end = (sp.sinks + KT - 1) / KT;
  a.first = sp.first;
  a.end = sp.end;
  return a;
}

// A piece of the share as the roles need it; one thread works ahead and leaves it in shared memory.
struct Piece {
  Seq s;
  Span span;
  Active act[2];
  int n;                                // key tiles v0 .. v0 + n; -1: there are no more pieces
  int v0, two, h, t_lo, tokens;
  int has[2];                           // whether a row tile (set of warps) sees any of them
  int whole;                            // the piece is the whole item
  int cut;                              // else: where its results go
};

struct Bars {
  uint64_t full[10], empty[10];         // ring
  uint64_t q_full, q_empty, dirty, fixed, drain, swap[2];
  uint64_t s_full[2], p_full[2], o_full[2], o_empty[2];
  uint64_t piece_full[2], piece_empty[2];
};
static_assert(sizeof(Bars) <= 512 && sizeof(Piece) <= 160, "the tail's layout");
constexpr int READERS = 2 + 1 + 8;      // of a piece: loads, tensor core, clearing warp, softmax warps

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

template <int D, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
attn_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_kv, const Batch p, const Outs w) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];                           // the swizzle wants it; nothing is left to align by hand
  uint8_t* q_s = smem;                                                        // [2][TILE]
  uint8_t* ring = smem + 2 * C::TILE;                                         // [STAGES][TILE]
  uint8_t* tail = ring + C::STAGES * C::TILE;
  Bars* bars = reinterpret_cast<Bars*>(tail);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 516);
  int* found = reinterpret_cast<int*>(tail + 520);                            // sequence, block
  long long* found_base = reinterpret_cast<long long*>(tail + 528);
  long long* wsum = reinterpret_cast<long long*>(tail + 544);                 // [12]
  int* wcnt = reinterpret_cast<int*>(tail + 640);                             // [12]
  float* ml = reinterpret_cast<float*>(tail + 704);                           // [2][MT][2]
  Piece* pieces = reinterpret_cast<Piece*>(tail + 2752);                      // [2]
  int* first_item = reinterpret_cast<int*>(ring);                             // [THREADS], before the first load
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tpt = MT / p.G;                                                   // tokens per row tile
  const int nb = p.a.B + p.b.B;

  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) { rb::mbar_init(&bars->full[i], 1); rb::mbar_init(&bars->empty[i], 1); }
    rb::mbar_init(&bars->q_full, 1); rb::mbar_init(&bars->q_empty, 1);
    rb::mbar_init(&bars->dirty, 1);
    rb::mbar_init(&bars->fixed, 32); rb::mbar_init(&bars->drain, 1);
    for (int i = 0; i < 2; ++i) {
      rb::mbar_init(&bars->s_full[i], 1); rb::mbar_init(&bars->p_full[i], MT);
      rb::mbar_init(&bars->o_full[i], 1); rb::mbar_init(&bars->o_empty[i], MT);
      rb::mbar_init(&bars->swap[i], 2 * MT);
      rb::mbar_init(&bars->piece_full[i], 1); rb::mbar_init(&bars->piece_empty[i], READERS);
    }
    *abort_flag = 0;
    rb::mbar_fence_init();
  }
  if (warp == 2) { rb::tmem_alloc(tmem_slot, 512); rb::tmem_relinquish(); }

  // ---- this CTA's share.  Blocks per sequence differ, so they are counted first and then dealt to the threads evenly.
  const int per = (nb + THREADS - 1) / THREADS;
  int n_mine = 0;
  for (int i = tid * per; i < min((tid + 1) * per, nb); ++i) n_mine += blocks_of(seq_of(p, i), tpt);
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
  // the sequence and block of item tid * ipt: the last thread whose first item is not after it owns it
  int seq0 = nb, blk0 = 0;
  const int my_first = tid * ipt, my_last = min(my_first + ipt, n_all);
  if (my_first < my_last) {
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
  auto each = [&](auto&& f) {                                                 // f(seq, block, units of all its items)
    int sq = seq0, bl = blk0;
    for (int i = my_first; i < my_last; ++i) {
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
  const int n_sh = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  Walk walk;
  walk.n_sh = n_sh; walk.total = total;
  walk.p0 = cta < n_sh ? share(cta, n_sh, total) : 0;
  walk.p1 = cta < n_sh ? share(cta + 1, n_sh, total) : 0;
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
  // the next piece, or null when there are no more (or a wait ran out; warps that work as one give up as one)
  auto next_piece = [&](bool as_warp) -> const Piece* {
    bool ok = !gave_up && rb::mbar_wait(&bars->piece_full[n_piece & 1], (n_piece >> 1) & 1, abort_flag, p.status, WAIT);
    if (as_warp) ok = __all_sync(0xffffffffu, ok);
    if (!ok) { gave_up = true; return nullptr; }
    const Piece* q = pieces + (n_piece & 1);
    return q->n < 0 ? nullptr : q;
  };
  auto done_piece = [&]() { rb::mbar_arrive(&bars->piece_empty[n_piece & 1]); ++n_piece; };

  if (warp == 3) {
    // ------------------------------------------------------------------ pieces
    if (lane == 0) {
      walk.seq = found[0]; walk.block = found[1]; walk.base = *found_base; walk.pos = walk.p0;
      if (walk.p0 >= walk.p1) walk.pos = walk.p1 = 0;
      Meta mt;
      mt.valid = 0;
      for (;; ++n_piece) {
        const bool more = walk.next(p, tpt);
        if (!rb::mbar_wait(&bars->piece_empty[n_piece & 1], ((n_piece >> 1) & 1) ^ 1, abort_flag, p.status, WAIT)) break;
        Piece& q = pieces[n_piece & 1];
        q.n = -1;
        if (more) {
          const Block& b = walk.b;
          q.s = walk.s; q.span = b.span; q.v0 = walk.v0(); q.n = max(walk.v1() - walk.v0(), 0); q.two = b.two; q.h = walk.h;
          q.t_lo = b.t_lo; q.tokens = b.tokens;
          for (int x = 0; x < 2; ++x) {
            const Active act = active_of(p, walk.s, b, x, tpt);
            q.act[x] = act;
            int has = !b.two && q.n > x;
            if (b.two) for (int j = 0; j < q.n && !has; ++j) has = act(b.span.tile(q.v0 + j));
            q.has[x] = has;
          }
          q.whole = walk.u0 == 0 && walk.u1 == b.units;
          q.cut = cta * 2 + (walk.pos == walk.p0 ? 0 : 1);
          const long long t0 = walk.pos - walk.u0;
          if (walk.pos == walk.p0 && walk.u0 > 0 && share(cta - 1, n_sh, total) <= t0) {
            // the first border inside this item: another kernel joins its pieces
            mt.valid = 1; mt.seq = walk.seq; mt.row0 = b.t_lo * p.G; mt.rows = b.tokens * p.G; mt.h = walk.h;
            mt.t0 = t0; mt.total = total; mt.n = n_sh; mt.c0 = cta - 1;
            mt.c1 = static_cast<int>(((t0 + b.units) * n_sh - 1) / total);
          }
          walk.done();
        }
        rb::mbar_arrive(&bars->piece_full[n_piece & 1]);
        if (!more) break;
      }
      w.meta[cta] = mt;
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------------ loads
    if (lane == 0) {
      int r = 0, n_q = 0;
      while (const Piece* q = next_piece(false)) {
        const bool two = q->two;
        const int v0 = q->v0, n = q->n, h = q->h;
        const Seq s = q->s;
        const Span sp = q->span;
        const int q_row = s.q_begin + q->t_lo;
        done_piece();
        if (n == 0) continue;
        auto load_kv = [&](int kind, int m) {                                 // kind 0: K, 1: V
          const int st = r % C::STAGES;
          if (gave_up || !rb::mbar_wait(&bars->empty[st], ((r / C::STAGES) & 1) ^ 1, abort_flag, p.status, WAIT)) { gave_up = true; return; }
          uint8_t* dst = ring + st * C::TILE;
          rb::mbar_expect_tx(&bars->full[st], C::TILE);
          const int k0 = sp.tile(v0 + m) * KT;
          for (int x = 0; x < KT; x += p.box_rows) {
            const int row = box_row(p, s, sp, k0 + x) + kind * p.page_size;
#pragma unroll
            for (int c = 0; c < C::CH; ++c)
              rb::tma_load_2d(dst + c * (KT * 128) + x * 128, &tm_kv, &bars->full[st], h * D + c * 64, row);
          }
          ++r;
        };
        if (!rb::mbar_wait(&bars->q_empty, (n_q & 1) ^ 1, abort_flag, p.status, WAIT)) { gave_up = true; break; }
        ++n_q;
        const int tiles_q = two ? 2 : 1;
        rb::mbar_expect_tx(&bars->q_full, tiles_q * C::CH * p.G * tpt * 128);
        for (int t = 0; t < tiles_q; ++t)
#pragma unroll
          for (int c = 0; c < C::CH; ++c)
            rb::tma_load_3d(q_s + t * C::TILE + c * (MT * 128), &tm_q, &bars->q_full, c * 64, h * p.G, q_row + t * tpt);
        // the order of k_index and v_index
        load_kv(0, 0);
        if (!two && n > 1) load_kv(0, 1);
        for (int m = 0; m < n; ++m) {
          load_kv(1, m);
          const int k = two ? m + 1 : m + 2;
          if (k < n) load_kv(0, k);
        }
      }
      if (gave_up)                                                            // copies in flight end before the kernel does
        for (int i = max(r - C::STAGES, 0); i < r; ++i)
          for (int k = 0; k < (1 << 16) && !rb::mbar_try_wait(&bars->full[i % C::STAGES], (i / C::STAGES) & 1); ++k) {}
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ tensor core
    if (lane == 0) {
      const uint32_t idesc_s = rb::umma_idesc(MT, KT, 0, 0, BF16), idesc_o = rb::umma_idesc(MT, D, 0, 1, BF16);
      const uint32_t q_addr = rb::smem_u32(q_s), ring_addr = rb::smem_u32(ring);
      int r0 = 0, n_q = 0, n_fix = 0;                                         // ring loads before this piece, blocks, cleared tiles
      uint32_t par_p = 0, par_o = 0;                                          // bit x: parity of row tile x's next P, next O
      while (const Piece* q = next_piece(false)) {
        const bool two = q->two;
        const int v0 = q->v0, n = q->n;
        const Span sp = q->span;
        const Active act0 = q->act[0], act1 = q->act[1];
        done_piece();
        if (n == 0) continue;
        const int slots = two ? n : (n + 1) / 2;
        int k_seen = -1, v_seen = -1;
        uint32_t started = 0;
        auto tile_at = [&](int slot, int x) { return two ? slot : 2 * slot + x; };
        auto valid = [&](int slot, int x) {
          const int m = tile_at(slot, x);
          if (slot >= slots || m >= n) return false;
          if (!two) return true;
          const int t = sp.tile(v0 + m);
          return x == 0 ? act0(t) : act1(t);
        };
        auto wait_full = [&](int idx) {
          if (!gave_up && !rb::mbar_wait(&bars->full[idx % C::STAGES], (idx / C::STAGES) & 1, abort_flag, p.status, WAIT)) gave_up = true;
          return !gave_up;
        };
        // a K or V tile is given back once its last user has been issued
        auto release = [&](int idx) { rb::umma_commit(&bars->empty[idx % C::STAGES]); };
        auto see_k = [&](int m) {
          if (m <= k_seen) return !gave_up;
          k_seen = m;
          return wait_full(r0 + k_index(two, m));
        };
        auto issue_s = [&](int slot, int x) {                                 // S_x = Q_x K^T
          const int m = tile_at(slot, x);
          if (!see_k(m)) return;
          rb::tc_fence_after();
          const uint32_t qa = q_addr + (two ? x : 0) * C::TILE, ka = ring_addr + ((r0 + k_index(two, m)) % C::STAGES) * C::TILE;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * (KT * 128) + (kk % 4) * 32;
            rb::umma_f16_ss(tmem + x * 128, rb::umma_smem_desc(qa + off, 16, 1024), rb::umma_smem_desc(ka + off, 16, 1024), idesc_s,
                            kk > 0 ? 1u : 0u);
          }
          rb::umma_commit(&bars->s_full[x]);
        };
        auto end_k = [&](int slot) {                                          // all of a slot's S are issued
          if (slot >= slots) return;
          for (int x = 0; x < (two ? 1 : 2); ++x) {
            const int m = tile_at(slot, x);
            if (m < n && see_k(m)) release(r0 + k_index(two, m));             // (a tile nobody needs has been loaded all the same)
          }
          if (slot == slots - 1) rb::umma_commit(&bars->q_empty);
        };
        if (!rb::mbar_wait(&bars->q_full, n_q & 1, abort_flag, p.status, WAIT)) { gave_up = true; break; }
        ++n_q;
        for (int x = 0; x < 2; ++x) if (valid(0, x)) issue_s(0, x);
        end_k(0);
        for (int j = 0; j < slots && !gave_up; ++j) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int m = tile_at(j, x);
            if (m < n && m > v_seen) {                                        // V of this tile, cleared where no row sees it
              v_seen = m;
              if (!wait_full(r0 + v_index(two, m, n))) break;
              const int k0 = sp.tile(v0 + m) * KT;
              if (!(k0 + KT <= sp.hi && (k0 >= sp.lo || k0 + KT <= sp.sinks))) {
                rb::mbar_arrive(&bars->dirty);
                if (!rb::mbar_wait(&bars->fixed, n_fix & 1, abort_flag, p.status, WAIT)) { gave_up = true; break; }
                ++n_fix;
              }
            }
            if (valid(j, x)) {
              const uint32_t bit = 1u << x;
              if (!(started & bit)) {
                if (!rb::mbar_wait(&bars->o_empty[x], ((par_o >> x) & 1) ^ 1, abort_flag, p.status, WAIT)) { gave_up = true; break; }
                par_o ^= bit;
              }
              if (!rb::mbar_wait(&bars->p_full[x], (par_p >> x) & 1, abort_flag, p.status, WAIT)) { gave_up = true; break; }
              par_p ^= bit;
              rb::tc_fence_after();
              const uint32_t va = ring_addr + ((r0 + v_index(two, m, n)) % C::STAGES) * C::TILE;
#pragma unroll
              for (int kk = 0; kk < KT / 16; ++kk)
                rb::umma_f16_ts(tmem + 256 + x * 128, tmem + x * 128 + kk * 8, rb::umma_smem_desc(va + kk * 2048, KT * 128, 1024), idesc_o,
                                ((started & bit) || kk > 0) ? 1u : 0u);
              started |= bit;
            }
            if (m < n && (!two || x == 1)) release(r0 + v_index(two, m, n));
            if (valid(j + 1, x)) issue_s(j + 1, x);
          }
          if (!gave_up) end_k(j + 1);
        }
        if (gave_up) break;
#pragma unroll
        for (int x = 0; x < 2; ++x) if (started & (1u << x)) rb::umma_commit(&bars->o_full[x]);
        r0 += 2 * n;
      }
      if (gave_up) {                                                          // nothing of ours still runs when TMEM is freed
        rb::umma_commit(&bars->drain);
        for (int k = 0; k < (1 << 16) && !rb::mbar_try_wait(&bars->drain, 0); ++k) {}
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ V rows that nobody sees
    int r0 = 0, n_fix = 0;
    while (const Piece* q = next_piece(true)) {
      const int v0 = q->v0, n = q->n;
      const bool two = q->two;
      const Span sp = q->span;
      __syncwarp();
      if (lane == 0) done_piece(); else ++n_piece;
      for (int m = 0; m < n && !gave_up; ++m) {
        const int k0 = sp.tile(v0 + m) * KT;
        if (k0 + KT <= sp.hi && (k0 >= sp.lo || k0 + KT <= sp.sinks)) continue;
        const bool ok = rb::mbar_wait(&bars->dirty, n_fix & 1, abort_flag, p.status, WAIT);      // it is there and still untouched
        if (!__all_sync(0xffffffffu, ok)) { gave_up = true; break; }
        ++n_fix;
        uint8_t* tile = ring + ((r0 + v_index(two, m, n)) % C::STAGES) * C::TILE;
        for (int i = lane; i < KT; i += 32) {
          const int j = k0 + i;
          if (j < sp.hi && (j >= sp.lo || j < sp.sinks)) continue;
          uint4* row = reinterpret_cast<uint4*>(tile + i * 128);
#pragma unroll
          for (int c = 0; c < C::CH; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) row[c * (KT * 8) + e] = make_uint4(0, 0, 0, 0);
        }
        rb::fence_proxy_async_smem();
        rb::mbar_arrive(&bars->fixed);
      }
      r0 += 2 * n;
    }
  } else {
    // ------------------------------------------------------------------ softmax: thread = row
    const int x = (warp - 4) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lane_sel + x * 128, t_o = tmem + lane_sel + 256 + x * 128;
    const int my_tok = row / p.G;                                              // of the row tile
    uint32_t par_s = 0, par_o = 0, par_swap = 0;
    while (const Piece* q = next_piece(true)) {
      const bool two = q->two;
      const int n = q->n;
      float m_ref = -INFINITY, sum = 0.f;                                      // log2 domain
      bool any = false;
      {
        const int v0 = q->v0, slots = two ? n : (n + 1) / 2;
        const Active act = q->act[x];
        const int sink_tiles = q->span.sink_tiles, skip = q->span.first - sink_tiles;
        const int len_k = q->s.len_k, causal = q->s.causal;
        const int pos = q->t_lo + (two ? x * tpt : 0) + my_tok + q->s.delta();
        // tiles that every row of the block sees in full: ends at or before p_min (hi), begins after p_max - window or is all sinks
        const int full_hi = causal ? q->span.p_min + 1 : q->span.hi;
        const int full_lo = causal && p.window > 0 ? q->span.p_max - p.window + 1 : 0;
        for (int j = 0; j < slots; ++j) {
          const int m = two ? j : 2 * j + x;
          if (m >= n) continue;
          const int t = v0 + m < sink_tiles ? v0 + m : v0 + m + skip;
          if (two && !act(t)) continue;
          const bool ok = rb::mbar_wait(&bars->s_full[x], par_s, abort_flag, p.status, WAIT);
          if (!__all_sync(0xffffffffu, ok)) { gave_up = true; break; }
          par_s ^= 1;
          rb::tc_fence_after();
          uint32_t sr[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) rb::tmem_ld_32x32(t_s + c * 32, sr[c]);
          rb::tmem_ld_wait();
          const int k0 = t * KT;
          if (!(k0 + KT <= full_hi && (k0 >= full_lo || k0 + KT <= p.sinks))) {
            // bit-wise limits of this row: keys below `upto`, of those from `from` on or sinks
            const int upto = min(causal ? min(pos + 1, len_k) : len_k, k0 + KT) - k0;
            const int from = causal && p.window > 0 ? pos - p.window + 1 - k0 : -1, sink = p.sinks - k0;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int i = c * 32 + e;
                if (i >= upto || (i < from && i >= sink)) sr[c][e] = 0xff800000u;
              }
          }
          float mx = -INFINITY, my = -INFINITY;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              mx = fmaxf(mx, __uint_as_float(sr[c][e]));
              my = fmaxf(my, __uint_as_float(sr[c][e + 1]));
            }
          const float m_new = fmaxf(mx, my) * p.scale_log2;                    // scale > 0 in this kernel
          // O and the sum refer to m_ref; only a row that outgrows it by 2^8 (or its first weight) moves it
          const bool grow = m_new > m_ref + 8.f || (m_ref == -INFINITY && m_new > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float f = grow ? (m_ref == -INFINITY ? 0.f : exp2_approx(m_ref - m_new)) : 1.f;
            if (grow) m_ref = m_new;
            sum *= f;
            if (any) {
              // S of this tile was issued after the product with the tile before: O is at rest
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
          for (int c = 0; c < 4; ++c) {
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
            rb::tmem_st_32x16(t_s + c * 16, pk);
          }
          sum = (acc0.x + acc0.y) + (acc1.x + acc1.y);
          rb::tmem_st_wait();
          rb::tc_fence_before();
          rb::mbar_arrive(&bars->p_full[x]);
          any = true;
        }
      }
      // ---- the piece's result: columns [c_lo, c_hi) of the row are this thread's to write
      int c_lo = 0, c_hi = D;
      float f0 = x == 0 ? 1.f : 0.f, f1 = 1.f - f0, l = sum, m_all = m_ref;
      const bool mine = q->has[x] != 0, theirs = q->has[x ^ 1] != 0;
      bool ok = !gave_up;
      if (!two) {
        ml[(x * MT + row) * 2] = m_ref; ml[(x * MT + row) * 2 + 1] = sum;
        rb::mbar_arrive(&bars->swap[0]);
        ok = rb::mbar_wait(&bars->swap[0], par_swap, abort_flag, p.status, WAIT) && ok;
        const float m0 = ml[row * 2], l0 = ml[row * 2 + 1], m1 = ml[(MT + row) * 2], l1 = ml[(MT + row) * 2 + 1];
        m_all = fmaxf(m0, m1);
        const float bm = m_all == -INFINITY ? 0.f : m_all;
        f0 = exp2_approx(m0 - bm); f1 = exp2_approx(m1 - bm);
        l = f0 * l0 + f1 * l1;
        c_lo = x * (D / 2); c_hi = c_lo + D / 2;
      }
      const bool read0 = two ? x == 0 && mine : q->has[0] != 0, read1 = two ? x == 1 && mine : q->has[1] != 0;
      if (ok && read0) ok = rb::mbar_wait(&bars->o_full[0], par_o & 1, abort_flag, p.status, WAIT);
      if (ok && read1) ok = rb::mbar_wait(&bars->o_full[1], (par_o >> 1) & 1, abort_flag, p.status, WAIT);
      if (!__all_sync(0xffffffffu, ok)) gave_up = true;
      rb::tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float lse2 = l == 0.f ? -INFINITY : m_all + log2f(l);
      f0 *= inv; f1 *= inv;
      if (!gave_up) {
        const int r_cut = two ? x * tpt * p.G + row : row;                      // row of the block
        const bool live = row < tpt * p.G && (two ? x * tpt : 0) + my_tok < q->tokens;
        const int row0 = q->t_lo * p.G, h = q->h;
        const bool whole = q->whole != 0;
        const long long cut = static_cast<long long>(q->cut) * TILE_ROWS + r_cut;
#pragma unroll 1
        for (int c = c_lo; c < c_hi; c += 16) {
          uint32_t a[16];
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
          if (read0) {
            rb::tmem_ld_32x16(tmem + lane_sel + 256 + c, a);
            rb::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = f0 * __uint_as_float(a[e]);
          }
          if (read1) {
            rb::tmem_ld_32x16(tmem + lane_sel + 384 + c, a);
            rb::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = fmaf(f1, __uint_as_float(a[e]), o[e]);
          }
          if (live) {
            if (whole) {
              write_row<D, BF16, 16>(p, w, q->s, row0 + r_cut, h, c, o, lse2);
            } else {
              float4* dst = reinterpret_cast<float4*>(w.cut_o + cut * D + c);
#pragma unroll
              for (int e = 0; e < 16; e += 4) dst[e >> 2] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
              if (c == 0) w.cut_lse[cut] = lse2;
            }
          }
        }
      }
      rb::tc_fence_before();
      if (!two) {                                                               // both sets of warps read both results
        rb::mbar_arrive(&bars->swap[1]);
        const bool both = rb::mbar_wait(&bars->swap[1], par_swap, abort_flag, p.status, WAIT);
        if (!__all_sync(0xffffffffu, both)) gave_up = true;
        par_swap ^= 1;
      }
      if (mine) { rb::mbar_arrive(&bars->o_empty[x]); par_o ^= 1u << x; }
      if (theirs) par_o ^= 1u << (x ^ 1);
      __syncwarp();
      if (lane == 0) done_piece(); else ++n_piece;
    }
  }
  __syncwarp();
  rb::tc_fence_before();
  __syncthreads();
  if (warp == 2) rb::tmem_dealloc(tmem, 512);
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
int launch(const Batch& p, const Outs& w, const void* cache, int n_cta, cudaStream_t st) {
  CUtensorMap tq, tkv;
  int rc = make_map_q(&tq, p, D, MT / p.G, BF16);
  if (rc) return rc;
  rc = rb_host::make_map_2d(&tkv, cache, p.total_rows, static_cast<long long>(p.Hkv) * D, static_cast<long long>(p.Hkv) * D, 64, p.box_rows, BF16);
  if (rc) return rc;
  RB_CUDA_CHECK(cudaFuncSetAttribute(attn_tiles_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM));
  attn_tiles_kernel<D, BF16><<<n_cta, THREADS, Cfg<D>::SMEM, st>>>(tq, tkv, p, w);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

int rb_attn::launch_tiles(const Batch& batch, const Outs& w, const void* cache, int D, bool is_bf16, int n_cta, cudaStream_t st) {
  Batch p = batch;
  p.box_rows = p.page_size % 64 == 0 ? 64 : p.page_size % 32 == 0 ? 32 : 16;
  if (D == 64) return is_bf16 ? launch<64, true>(p, w, cache, n_cta, st) : launch<64, false>(p, w, cache, n_cta, st);
  return is_bf16 ? launch<128, true>(p, w, cache, n_cta, st) : launch<128, false>(p, w, cache, n_cta, st);
}
