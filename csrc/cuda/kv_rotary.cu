// Appending keys and values to the paged KV cache with the position rotation applied on the way (sm_100a).
//
//   (x_a, x_b) -> (x_a c - x_b s, x_b c + x_a s)    c, s = table[position][i], table[position][R/2 + i],  i < R/2
//
// for the R leading elements of every query and key head; (a, b) = (i, i + R/2), or (2i, 2i + 1) when interleaved.  The
// rest of a head and all of V are copied.  K and V go straight into their pages [pages][2][page][Hkv*D], the turned
// queries into a tensor of their own, so each of the three is read and written once.
//
// Bound: memory.  A unit of work is 16 elements of a head (two 16-byte loads whose elements turn with each other, so no
// exchange between threads), and one thread takes the same unit of up to four heads of a token: the eight loads are in
// flight together and the unit's cosines and sines (64 bytes of the fp32 table) are read once for them.
// 20011 tokens, 32 + 2 x 8 heads of 128: 0.5 GB in 89 to 94 us, 81 to 85 % of a copy's bandwidth; a single token: 3.6 us in a graph, the launch.
#include "common.cuh"

namespace {

constexpr int HPT = 4;    // heads per thread

struct RotaryArgs {
  const uint16_t *q, *k, *v;
  long long ld_q, ld_k, ld_v;        // elements between tokens; heads of a token are adjacent
  uint16_t* q_out; long long ld_o;
  uint16_t* cache;
  const int *batch_idx, *positions, *page_ids, *page_indptr;
  const int* slots;                  // place among the request's tokens, or null: its position
  const int* num_tokens;             // device [1] or null: tokens at or past it are left alone
  int nnz, H, Hkv, D, B, page_size, num_page_ids;
  long long num_pages;
  const float* table; int table_rows, R;
  int interleaved;
  int* status;
};

template <bool BF16> __device__ __forceinline__ float2 unpack(uint32_t u) { return BF16 ? rb::unpack_bf16(u) : rb::unpack_f16(u); }
template <bool BF16> __device__ __forceinline__ uint32_t pack(float a, float b) { return BF16 ? rb::pack_bf16(a, b) : rb::pack_f16(a, b); }

// fp32 products of the 16-bit values with the table, rounded to 16 bits once
template <bool BF16>
__device__ __forceinline__ void turn(uint4& a, uint4& b, const float (&c)[8], const float (&s)[8], bool interleaved) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
  uint32_t* pb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (interleaved) {
      const float2 x = unpack<BF16>(pa[w]), y = unpack<BF16>(pb[w]);
      pa[w] = pack<BF16>(x.x * c[w] - x.y * s[w], x.y * c[w] + x.x * s[w]);
      pb[w] = pack<BF16>(y.x * c[w + 4] - y.y * s[w + 4], y.y * c[w + 4] + y.x * s[w + 4]);
    } else {
      const float2 x = unpack<BF16>(pa[w]), y = unpack<BF16>(pb[w]);
      pa[w] = pack<BF16>(x.x * c[2 * w] - y.x * s[2 * w], x.y * c[2 * w + 1] - y.y * s[2 * w + 1]);
      pb[w] = pack<BF16>(y.x * c[2 * w] + x.x * s[2 * w], y.y * c[2 * w + 1] + x.y * s[2 * w + 1]);
    }
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256) kv_append_rotary_kernel(const RotaryArgs p) {
  const int units = p.D >> 4, heads = p.H + 2 * p.Hkv;
  const int slots = (heads + HPT - 1) / HPT;
  const int per_token = slots * units;
  const int n = p.num_tokens ? min(p.nnz, max(*p.num_tokens, 0)) : p.nnz;
  const long long total = static_cast<long long>(n) * per_token;
  for (long long e = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; e < total;
       e += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int i = static_cast<int>(e / per_token);
    const int r = static_cast<int>(e - static_cast<long long>(i) * per_token);
    const int slot = r / units, u = r - slot * units;
    const bool rotary = u < (p.R >> 4);
    const int va = (rotary && !p.interleaved) ? u : 2 * u;                   // the unit's two vectors of 8 elements
    const int vb = (rotary && !p.interleaved) ? u + (p.R >> 4) : 2 * u + 1;
    uint4 a[HPT], b[HPT];
#pragma unroll
    for (int t = 0; t < HPT; ++t) {
      const int h = slot + t * slots;
      if (h >= heads) continue;
      const uint16_t* src = h < p.H ? p.q + i * p.ld_q + h * p.D
                            : h < p.H + p.Hkv ? p.k + i * p.ld_k + (h - p.H) * p.D
                                              : p.v + i * p.ld_v + (h - p.H - p.Hkv) * p.D;
      a[t] = reinterpret_cast<const uint4*>(src)[va];                        // (no __ldg: q_out may be q)
      b[t] = reinterpret_cast<const uint4*>(src)[vb];
    }
    const int pos = p.positions[i], at_token = p.slots ? p.slots[i] : pos, bi = p.batch_idx[i];
    bool ok = pos >= 0 && pos < p.table_rows && at_token >= 0 && bi >= 0 && bi < p.B;
    long long page = 0;
    if (ok) {
      const long long at = static_cast<long long>(p.page_indptr[bi]) + at_token / p.page_size;
      ok = at >= 0 && at < p.page_indptr[bi + 1] && at < p.num_page_ids;
      if (ok) {
        page = p.page_ids[at];
        ok = page >= 0 && page < p.num_pages;
      }
    }
    if (!ok) {                                                               // reported; nothing of the token is written
      if (p.status) atomicCAS(p.status, 0, RB_ERR_BOUNDS);
      continue;
    }
    float c[8], s[8];
    if (rotary) {
      const float4* row = reinterpret_cast<const float4*>(p.table + static_cast<long long>(pos) * p.R);
      const float4 c0 = __ldg(row + 2 * u), c1 = __ldg(row + 2 * u + 1);
      const float4 s0 = __ldg(row + (p.R >> 3) + 2 * u), s1 = __ldg(row + (p.R >> 3) + 2 * u + 1);
      c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
      s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
    }
    const long long row_elems = static_cast<long long>(p.Hkv) * p.D;
    uint16_t* k_row = p.cache + ((page * 2) * p.page_size + at_token % p.page_size) * row_elems;
#pragma unroll
    for (int t = 0; t < HPT; ++t) {
      const int h = slot + t * slots;
      if (h >= heads) continue;
      uint16_t* dst = h < p.H ? p.q_out + i * p.ld_o + h * p.D
                      : h < p.H + p.Hkv ? k_row + (h - p.H) * p.D
                                        : k_row + p.page_size * row_elems + (h - p.H - p.Hkv) * p.D;
      if (rotary && h < p.H + p.Hkv) turn<BF16>(a[t], b[t], c, s, p.interleaved != 0);
      reinterpret_cast<uint4*>(dst)[va] = a[t];
      reinterpret_cast<uint4*>(dst)[vb] = b[t];
    }
  }
}

}  // namespace

// The arguments of rb_kv_append_rotary, 8-byte fields first (the caller packs them).
// q [nnz][H][D], k / v [nnz][Hkv][D] 16-bit (bf16 or fp16), token strides in elements (multiples of 8, 16-byte aligned
// bases); cache [num_pages][2][page_size][Hkv*D]; table [table_rows][R] fp32 = R/2 cosines, R/2 sines; D and R multiples of
// 16, R <= D.  slots [nnz] or null, num_tokens: device [1] or null.  A token whose position, batch index or page is out of range is skipped and
// reported in status.
struct KvAppendCall {
  const void* q; long long ld_q; const void* k; long long ld_k; const void* v; long long ld_v;
  void* q_out; long long ld_o;
  void* cache; long long num_pages;
  const int *batch_idx, *positions, *slots, *page_ids, *page_indptr, *num_tokens;
  const float* table;
  int* status; cudaStream_t stream;
  int nnz, H, Hkv, D, B, page_size, num_page_ids, table_rows, R, interleaved, is_bf16, num_sms;
};

RB_API int rb_kv_append_rotary(const void* call) {
  const KvAppendCall& c = *static_cast<const KvAppendCall*>(call);
  if (c.nnz == 0) return 0;
  if (c.D % 16 || c.R % 16 || c.R <= 0 || c.R > c.D || c.page_size <= 0) return -1;
  if (c.ld_q % 8 || c.ld_k % 8 || c.ld_v % 8 || c.ld_o % 8) return -2;
  RotaryArgs p;
  p.q = (const uint16_t*)c.q; p.k = (const uint16_t*)c.k; p.v = (const uint16_t*)c.v; p.ld_q = c.ld_q; p.ld_k = c.ld_k; p.ld_v = c.ld_v;
  p.q_out = (uint16_t*)c.q_out; p.ld_o = c.ld_o; p.cache = (uint16_t*)c.cache; p.batch_idx = c.batch_idx; p.positions = c.positions;
  p.slots = c.slots; p.page_ids = c.page_ids; p.page_indptr = c.page_indptr; p.num_tokens = c.num_tokens; p.nnz = c.nnz; p.H = c.H; p.Hkv = c.Hkv; p.D = c.D;
  p.B = c.B; p.page_size = c.page_size; p.num_page_ids = c.num_page_ids; p.num_pages = c.num_pages; p.table = c.table;
  p.table_rows = c.table_rows; p.R = c.R; p.interleaved = c.interleaved; p.status = c.status;
  const long long work = static_cast<long long>(c.nnz) * ((c.H + 2 * c.Hkv + HPT - 1) / HPT) * (c.D / 16);
  const long long cap = static_cast<long long>(c.num_sms > 0 ? c.num_sms : 148) * 8 * 8;
  long long blocks = (work + 255) / 256;
  if (blocks > cap) blocks = cap;
  if (c.is_bf16) kv_append_rotary_kernel<true><<<static_cast<int>(blocks), 256, 0, c.stream>>>(p);
  else kv_append_rotary_kernel<false><<<static_cast<int>(blocks), 256, 0, c.stream>>>(p);
  return static_cast<int>(cudaGetLastError());
}
