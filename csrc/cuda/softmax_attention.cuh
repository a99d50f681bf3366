// What the softmax-attention kernels over the paged KV cache share: the description of a batch, which keys a block of
// query rows sees, and how their partial results are laid out.
#pragma once
#include "common.cuh"

namespace rb_attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// One list of sequences whose keys live in pages.  A query row is (token, head); the rows of the G = H / Hkv heads that
// share a key head are packed: row r of a sequence is token r / G, head r % G of the group.
struct Seqs {
  const int* q_offsets;       // [B+1] rows of q per sequence ...
  const int* group_offsets;   // ... or null; [B+1] into q_offsets: sequence g holds the queries of requests go[g]..go[g+1]-1
  int one_group;              // B is 1 and holds the queries of all requests
  const int* k_offsets;       // [B+1] keys per sequence (differences are used)
  const int* page_ids;
  const int* page_indptr;     // [B+1]
  int num_page_ids;
  int B;
  int num_requests;           // q_offsets has num_requests + 1 entries
  int causal;                 // a row sees the keys up to its own position; 0: all of them
};

struct Batch {
  Seqs a, b;                  // sequences of b (may be none) are numbered after those of a
  const void* q; long long ld_q;
  int Tq, H, Hkv, G;
  int page_size, box_rows, total_rows;   // of the cache as a matrix [pages * 2 * page_size][Hkv * D]
  int window, sinks;          // window 0: no limit
  float scale_log2;           // scale * log2(e)
  int* status;
};

struct Seq {
  int q_begin, len_q, len_k, page_begin, page_end, causal, part;
  const int* page_ids;
  __device__ __forceinline__ int delta() const { return len_k - len_q; }
};

__device__ __forceinline__ Seq seq_of(const Batch& p, int i) {
  const bool second = i >= p.a.B;
  const Seqs& s = second ? p.b : p.a;
  const int j = second ? i - p.a.B : i;
  Seq r;
  int q0 = j, q1 = s.one_group ? s.num_requests : j + 1;
  if (s.group_offsets) {
    q0 = min(max(s.group_offsets[j], 0), s.num_requests);
    q1 = min(max(s.group_offsets[j + 1], q0), s.num_requests);
  }
  // rows outside q are never touched, whatever the offsets say
  r.q_begin = min(max(s.q_offsets[q0], 0), p.Tq);
  r.len_q = min(max(s.q_offsets[q1], r.q_begin), p.Tq) - r.q_begin;
  // (the offsets may have passed 32 bits: their difference is the same)
  r.len_k = max(static_cast<int>(static_cast<unsigned>(s.k_offsets[j + 1]) - static_cast<unsigned>(s.k_offsets[j])), 0);
  r.page_begin = min(max(s.page_indptr[j], 0), s.num_page_ids);               // (so that no page's number passes 32 bits)
  r.page_end = min(s.page_indptr[j + 1], s.num_page_ids);
  r.page_ids = s.page_ids;
  r.causal = s.causal;
  r.part = second ? 1 : 0;
  return r;
}

// Keys that a block of consecutive rows may see, in tiles of T keys aligned to multiples of T: first the tiles that hold
// sinks, then the tiles of the window.
struct Span {
  int p_min, p_max;           // positions of the first and the last token of the block
  int hi;                     // keys at or past it are seen by no row of the block
  int lo;                     // keys before it are seen by no row, unless they are sinks
  int sinks;
  int sink_tiles, first, end, tiles;   // tile v is v < sink_tiles ? v : first + v - sink_tiles
  __device__ __forceinline__ int tile(int v) const { return v < sink_tiles ? v : first + v - sink_tiles; }
};

template <int T>
__device__ __forceinline__ Span span_of(const Batch& p, const Seq& s, int t_lo, int t_hi) {
  Span r;
  const int delta = s.delta();
  r.p_min = s.causal ? t_lo + delta : s.len_k - 1;
  r.p_max = s.causal ? t_hi + delta : s.len_k - 1;
  r.hi = max(min(s.len_k, r.p_max + 1), 0);
  const bool win = s.causal && p.window > 0;
  r.lo = win ? max(r.p_min - p.window + 1, 0) : 0;
  r.sinks = win ? min(p.sinks, r.hi) : 0;
  r.end = (r.hi + T - 1) / T;
  r.first = r.lo / T;
  r.sink_tiles = min((r.sinks + T - 1) / T, r.first);
  r.tiles = r.sink_tiles + max(r.end - r.first, 0);
  return r;
}

// Which of the keys j0 .. j0 + 31 the row at position pos sees: bit i for key j0 + i
__device__ __forceinline__ uint32_t seen_keys(int pos, int j0, int len_k, int causal, int window, int sinks) {
  auto below = [&](int n) { const int d = n - j0; return d >= 32 ? 0xffffffffu : d <= 0 ? 0u : (1u << d) - 1u; };
  uint32_t seen = below(causal ? min(pos + 1, len_k) : len_k);
  if (causal && window > 0) seen &= ~below(pos - window + 1) | below(sinks);
  return seen;
}

// Row of the cache matrix where the box of keys j.. starts (K; V is page_size rows further), or a row past the end, which
// a TMA load fills with zeros: for boxes of keys that no row of the block sees, whose pages may be gone, and - reported -
// for pages that are not there.
__device__ __forceinline__ int box_row(const Batch& p, const Seq& s, const Span& r, int j) {
  if (j >= r.hi || (j + p.box_rows <= r.lo && j >= r.sinks)) return p.total_rows;
  const int at = s.page_begin + j / p.page_size;
  const int per_page = 2 * p.page_size;
  if (at < s.page_end) {
    const int page = __ldg(s.page_ids + at);
    if (page >= 0 && page < p.total_rows / per_page) return page * per_page + j % p.page_size;
  }
  if (p.status) atomicCAS(p.status, 0, RB_ERR_BOUNDS);
  return p.total_rows;
}

// log2 of the largest weight that is handed to the product with V, which takes weights in the inputs' type: bf16 has fp32's
// exponents and may have it anywhere, fp16's range ends just above 2^15.
template <bool BF16> constexpr float WeightTop = BF16 ? 0.f : 15.f;

template <bool BF16> __device__ __forceinline__ uint32_t pack16(float a, float b) { return BF16 ? rb::pack_bf16(a, b) : rb::pack_f16(a, b); }

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The keys of all items (sequence, block of rows, key head) are laid end to end in units and cut into as many equal shares as
// there are workers; none is empty.
struct Shares {
  long long total, q;                      // q = total / n
  uint32_t r;                              // total % n
  int n;
  __device__ __forceinline__ Shares(long long units, int workers) : total(units), n(static_cast<int>(min(static_cast<long long>(workers), units))) {
    q = n ? units / n : 0;                 // the one division of 64 bits
    r = static_cast<uint32_t>(units - q * n);
  }
  // floor(total * c / n): where share c begins
  __device__ __forceinline__ long long begin(int c) const { return c < n ? q * c + r * static_cast<uint32_t>(c) / static_cast<uint32_t>(n) : total; }
  // the share that holds a unit
  __device__ __forceinline__ int of(long long unit) const { return static_cast<int>(((unit + 1) * n - 1) / total); }
};

// Rows [row0, row0 + rows) of a sequence (packed: token * G + head of the group) whose units shares c0..c1 hold; left by
// the share c0 + 1 for the kernel that joins the pieces.
struct Meta { int valid, seq, row0, rows, h, c0, c1, first; };   // first: piece c0's place, 2 * c0 or 2 * c0 + 1

struct Outs {
  void* out; long long ld_o; float* lse;   // final results: 16-bit rows [Tq][ld_o], lse [Tq][H] or null
  float* part_o; float* part_lse;          // when not null: fp32 [2][Tq][H][D] and log2 [2][Tq][H] instead, by Seq::part
  float* cut_o; float* cut_lse;            // [shares][2][rows of a block][D], [shares][2][rows]: pieces of items cut by a border
  Meta* meta;                              // [shares]
};

// Where a row's result goes: 16 bits to the output, or fp32 to its part or to its place among the cut pieces
struct RowOut { uint16_t* o16; float* o32; float* lse; int natural; };   // natural: lse to base e, else log2

__device__ __forceinline__ RowOut row_out(const Batch& p, const Outs& w, const Seq& s, int row, int h, int D, bool whole, long long cut) {
  RowOut r = {nullptr, nullptr, nullptr, 0};
  const long long t = s.q_begin + row / p.G;
  const int head = h * p.G + row % p.G;
  if (!whole) {
    r.o32 = w.cut_o + cut * D;
    r.lse = w.cut_lse + cut;
  } else if (w.part_o) {
    const long long at = (static_cast<long long>(s.part) * p.Tq + t) * p.H + head;
    r.o32 = w.part_o + at * D;
    r.lse = w.part_lse + at;
  } else {
    r.o16 = reinterpret_cast<uint16_t*>(w.out) + t * w.ld_o + static_cast<long long>(head) * D;
    r.lse = w.lse ? w.lse + t * p.H + head : nullptr;
    r.natural = 1;
  }
  return r;
}

// softmax_attention_tiles.cu: the kernel for many rows per sequence; fills out / part and the cut pieces (blocks of
// TILE_ROWS rows) of all sequences of p
constexpr int TILE_ROWS = 256;
int launch_tiles(const Batch& p, const Outs& w, const void* cache, int D, bool is_bf16, int n_cta, bool after, cudaStream_t st);

// The kernels of a call follow one another with programmatic launches: each lets the next one start early, and the next
// one waits (for the whole of what ran before, and by that for what ran before that) where it needs its results.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// `after`: not the first kernel of a call (that one is ordered behind the caller's work as usual)
template <typename... P, typename... A>
int launch_kernel(bool after, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = after ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, static_cast<A&&>(args)...));
}

}  // namespace rb_attn
