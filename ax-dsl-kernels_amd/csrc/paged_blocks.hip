// Sparse attention over a paged KV cache, and eviction of its pages, for gfx950.
//
// A page of the cache (layout and page table as in paged_attn.hip) is cut into blocks of `block` consecutive tokens
// (block a multiple of 16 that divides the page). For every block and KV head, bounds[P, page / block, HKV, 2, D]
// (bf16) keeps the channel-wise minimum and maximum of the block's keys, rounded outward where bf16 does not hold them
// (int8 caches). One decode step is then
//   1. paged_kv_write_bounds_kernel  the new tokens' K / V into the cache and into their blocks' bounds
//      (paged_key_bounds_kernel      the bounds from the cache: after a prefill chunk, or for a whole cache)
//   2. paged_block_scores_kernel     s[h, j] = max_g sum_d max(q_gd lo_jd, q_gd hi_jd), which no q_g . k of block j exceeds
//   3. paged_select_blocks_kernel    the n best blocks of each (sequence, KV head), in ascending order
//   4. paged_blocks_kernel, paged_blocks_merge_kernel   attention over those blocks (or all of them), and each page's
//                                    share of it, w_out = decay w_in + sum over the KV head's queries
// and, when a sequence has grown past its budget,
//   5. paged_evict_kernel            the page table without the pages of least w.
#include <math.h>

#include "axk_common.h"
#include "axk_host.h"

namespace {

constexpr int kSub = 16;       // tokens of a subtile: the rows of one MFMA operand, and the unit of the block size
constexpr int kMaxGroup = 16;  // query heads per KV head (the other side of that operand)
constexpr float kLog2e = 1.4426950408889634f;

// Sequence b of a page table with nnz entries: its first entry, its pages and its tokens. Offsets outside the table and
// a last page longer than a page are clamped, so that no index built from them leaves its array.
struct Seq {
  int pb, np;
  int64_t len;
};
AXK_DEV Seq seq_from(int lo, int hi, int last, int page, int nnz) {
  Seq s;
  s.pb = min(max(lo, 0), nnz);
  s.np = min(max(hi, s.pb), nnz) - s.pb;
  s.len = s.np ? (int64_t)(s.np - 1) * page + min(max(last, 0), page) : 0;
  return s;
}
// Its subtiles of 16 tokens, and blocks: 32 bits, as all that is divided here (a 64-bit division is some 130 instructions).
AXK_DEV int subs_of(const Seq& s) { return (int)((s.len + kSub - 1) / kSub); }
AXK_DEV int blocks_of(const Seq& s, int block) { return (int)((unsigned)(subs_of(s) + block / kSub - 1) / (unsigned)(block / kSub)); }
AXK_DEV Seq seq_of(const int* __restrict__ indptr, const int* __restrict__ last, int b, int page, int nnz) {
  return seq_from(indptr[b], indptr[b + 1], last[b], page, nnz);
}

// The sequence that holds page-table entry e (b = batch: none does), found by one wave: lanes hold 64 sequences at a time,
// so that up to 64 sequences cost one round trip to memory, with the sequence's own numbers.
struct Owner {
  int b;
  Seq s;
};
AXK_DEV Owner owner_of(const int* __restrict__ indptr, const int* __restrict__ last, int batch, int page, int nnz, int e) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int b = min(b0 + lane, batch - 1);
    const int lo = indptr[b], hi = indptr[b + 1], tail = last[b];
    const uint64_t after = __ballot(hi > e);  // sequences ending past e: the first of them
    if (after) {
      const int src = __ffsll((unsigned long long)after) - 1;
      return {b0 + src, seq_from(__builtin_amdgcn_readlane(lo, src), __builtin_amdgcn_readlane(hi, src),
                                 __builtin_amdgcn_readlane(tail, src), page, nnz)};
    }
  }
  return {batch, {0, 0, 0}};
}

// Inclusive sum over the lanes of a wave: shifts within rows of 16 lanes, then the rows' totals passed on.
AXK_DEV unsigned wave_scan(unsigned v) {
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
  return v;
}
AXK_DEV int wave_total(int v) { return __builtin_amdgcn_readlane((int)wave_scan((unsigned)v), 63); }

// Two bf16 values (one dword) as two 16-bit integers of the same order, and back (the map is its own inverse): the 15
// low bits of a negative value are flipped. NaN lies beyond the infinity of its sign.
typedef short axk_s16x2 __attribute__((ext_vector_type(2)));
AXK_DEV axk_s16x2 bf16_order(uint32_t w) {
  const axk_s16x2 x = __builtin_bit_cast(axk_s16x2, w);
  return x ^ ((x >> (short)15) & (short)0x7fff);
}
AXK_DEV uint32_t bf16_unorder(axk_s16x2 x) { return __builtin_bit_cast(uint32_t, x ^ ((x >> (short)15) & (short)0x7fff)); }

// What a cache stores: bf16; E4M3 bytes, attended as stored * inv_scale (a power of two: exact in bf16); or int8 codes with a
// bf16 scale per row and KV head, attended as code * scale.
enum { kBf16 = 0, kFp8 = 1, kI8 = 2 };

// Byte i of w, an int8 code, as a float.
AXK_DEV float i8_code(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }
// A dword of stored 8-bit values as two bf16 pairs (int8: the codes, exact in bf16).
template <int T>
AXK_DEV uint32_t pair_of(uint32_t w, int hi, float inv_scale) {
  if constexpr (T == kI8) return pack_bf16x2(i8_code(w, 2 * hi), i8_code(w, 2 * hi + 1));
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, inv_scale, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, inv_scale, false));
}
// An int8 key, code * scale, has up to 16 significant bits and is attended unrounded, so its bf16 bounds are rounded
// outward: x down and up to bf16, in the high half of a dword (a magnitude's low half carries into the high one where the
// value moves away from zero). NaN goes past the infinity of either side.
AXK_DEV uint32_t bf16_down(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0xffff0000u : u + ((uint32_t)((int)u >> 31) >> 16);
}
AXK_DEV uint32_t bf16_up(float x) {
  const uint32_t u = __float_as_uint(x);
  return x != x ? 0x7fff0000u : u + (~(uint32_t)((int)u >> 31) >> 16);
}
AXK_DEV uint32_t high_halves(uint32_t x, uint32_t y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); }

// 16 bytes of stored keys as bf16 pairs in order: 4 dwords of a bf16 cache, 8 of an 8-bit one.
template <int T>
AXK_DEV void stored_pairs(const axk_u32x4 w, float inv_scale, uint32_t (&out)[T ? 8 : 4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T) {
      out[2 * i] = pair_of<T>(w[i], 0, inv_scale);
      out[2 * i + 1] = pair_of<T>(w[i], 1, inv_scale);
    } else {
      out[i] = w[i];
    }
  }
}

// ---- key bounds ----
constexpr int64_t kMaxRows = 16384;  // every row looks at every other's place: 16384 rows take 0.22 ms, 1024 10.6 us

// The new rows' K / V written at loc[r] = (page, slot), and folded into the bounds of their blocks: a block that holds a
// new row at its first slot starts afresh, every other one widens what it had. One workgroup per row; the first row of
// the call that falls into a block folds all of them, so that rows of one block never race, and where two rows name one
// slot the last one is stored (both are folded). Bound by its chain: launch, locations, then row and bounds; 3.4 us for the
// 16 rows of a decode step (HKV 2, D 256), 2.3 without the bounds, 4.5 for 16 rows of one block; into an int8 cache 4.7 and
// 14.5, as a row is quantized once for the cache and once for the bounds.
//
// Eight channels of a new row as the cache keeps them: their bytes (a bf16 cache: the values themselves), the int8 scale,
// and the key's bf16 pairs as attention reads them, rounded down and up where they have more bits (int8). The d / 8 lanes of
// a head's row act together.
struct Stored {
  uint32_t lo, hi;            // 8-bit caches: the eight bytes
  float scale;                // int8
  uint32_t down[4], up[4];
};
template <int T>
AXK_DEV Stored store_eight(const uint4 src, int d, float kv_scale) {
  const uint32_t w[4] = {src.x, src.y, src.z, src.w};
  Stored o = {0u, 0u, 0.f, {w[0], w[1], w[2], w[3]}, {w[0], w[1], w[2], w[3]}};
  if constexpr (T == kBf16) return o;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(e & 1 ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
  float r = 0.f;
  if constexpr (T == kI8) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
    for (int m = d / 16; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));  // the row's lanes: d / 8, aligned
    o.scale = kv_i8_scale(amax);
    r = round_bf16(1.0f / o.scale);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t c = T == kFp8 ? f32_to_e4m3(round_bf16(x[e] * kv_scale)) : ((uint32_t)(int)kv_i8_code(x[e], r) & 0xffu);
    if (e < 4) o.lo |= c << (8 * e); else o.hi |= c << (8 * (e - 4));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = i < 2 ? o.lo : o.hi;
    if constexpr (T == kI8) {
      const float y0 = i8_code(b, 2 * (i & 1)) * o.scale, y1 = i8_code(b, 2 * (i & 1) + 1) * o.scale;
      o.down[i] = high_halves(bf16_down(y0), bf16_down(y1));
      o.up[i] = high_halves(bf16_up(y0), bf16_up(y1));
    } else {
      o.down[i] = o.up[i] = pair_of<T>(b, i & 1, 1.0f / kv_scale);
    }
  }
  return o;
}

template <int T>
__global__ __launch_bounds__(256) void paged_kv_write_bounds_kernel(
    const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, unsigned char* __restrict__ cache,
    uint16_t* __restrict__ scales, uint16_t* __restrict__ bounds, const int* __restrict__ loc, int rows, int hkv, int d,
    int page_size, int block, int64_t num_pages, float kv_scale, int* __restrict__ status) {
  __shared__ int s_rows[256];
  __shared__ int s_count, s_first, s_fresh, s_over;
  const int tid = threadIdx.x, r = blockIdx.x;
  const int page = loc[2 * r], off = loc[2 * r + 1];
  if (page < 0 || page >= num_pages || off < 0 || off >= page_size) {
    if (status && tid == 0) *status = 1;
    return;
  }
  if (tid == 0) {
    s_first = 1;
    s_fresh = 0;
    s_over = 0;
  }
  __syncthreads();
  const int blk = off / block;
  // which rows of the call share the block: an earlier one owns it, a later one at the same slot is the one stored
  for (int i = tid; i < rows; i += 256) {
    const int p = loc[2 * i], o = loc[2 * i + 1];
    if (p != page || o < 0 || o >= page_size || o / block != blk) continue;
    if (i < r) s_first = 0;
    if (o % block == 0) s_fresh = 1;
    if (i > r && o == off) s_over = 1;
  }
  __syncthreads();
  const int row = hkv * d, chunks = row / 8;  // values of one token row, and its pieces of 8 channels
  if (!s_over) {
    for (int i = tid; i < 2 * chunks; i += 256) {
      const int plane = i >= chunks, ch = plane ? i - chunks : i;
      const uint4 src = *reinterpret_cast<const uint4*>((plane ? v : k) + (int64_t)r * row + ch * 8);
      const int64_t slot = ((int64_t)page * 2 + plane) * page_size + off, at = slot * row + ch * 8;
      if constexpr (T == kBf16) {
        *reinterpret_cast<uint4*>(cache + 2 * at) = src;
      } else {
        const Stored o = store_eight<T>(src, d, kv_scale);
        *reinterpret_cast<uint2*>(cache + at) = make_uint2(o.lo, o.hi);
        if (T == kI8 && ch * 8 % d == 0) scales[slot * hkv + ch * 8 / d] = (uint16_t)f32_to_bf16_bits(o.scale);
      }
    }
  }
  if (!s_first) return;
  const int fresh = s_fresh;
  uint16_t* bb = bounds + ((int64_t)page * (page_size / block) + blk) * hkv * 2 * d;
  for (int base = r & ~255; base < rows; base += 256) {  // the call's rows from this one on, 256 at a time
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
    const int i = base + tid;
    if (i >= r && i < rows) {
      const int p = loc[2 * i], o = loc[2 * i + 1];
      if (p == page && o >= 0 && o < page_size && o / block == blk) s_rows[atomicAdd(&s_count, 1)] = i;
    }
    __syncthreads();
    const int n = s_count;
    for (int c = tid; n && c < chunks; c += 256) {  // 8 channels of one head at a time
      const int head = c * 8 / d, ch = c * 8 - head * d;
      uint16_t* lo_p = bb + (int64_t)head * 2 * d + ch;
      uint4* lo4 = reinterpret_cast<uint4*>(lo_p);
      uint4* hi4 = reinterpret_cast<uint4*>(lo_p + d);
      axk_s16x2 lo[4], hi[4];
      const bool from = !fresh || base > r;  // the bounds already there count (the list's first row has index >= r)
      const uint4 l0 = *lo4, h0 = *hi4;
      const uint32_t lw[4] = {l0.x, l0.y, l0.z, l0.w}, hw[4] = {h0.x, h0.y, h0.z, h0.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = from ? bf16_order(lw[e]) : (axk_s16x2)(short)0x7fff;
        hi[e] = from ? bf16_order(hw[e]) : (axk_s16x2)(short)-0x8000;
      }
      for (int j0 = 0; j0 < n; j0 += 8) {  // eight rows' loads under way together
        uint4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j0 + j < n) x[j] = *reinterpret_cast<const uint4*>(k + (int64_t)s_rows[j0 + j] * row + c * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j0 + j >= n) break;
          const Stored o = store_eight<T>(x[j], d, kv_scale);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            lo[e] = __builtin_elementwise_min(lo[e], bf16_order(o.down[e]));
            hi[e] = __builtin_elementwise_max(hi[e], bf16_order(o.up[e]));
          }
        }
      }
      *lo4 = make_uint4(bf16_unorder(lo[0]), bf16_unorder(lo[1]), bf16_unorder(lo[2]), bf16_unorder(lo[3]));
      *hi4 = make_uint4(bf16_unorder(hi[0]), bf16_unorder(hi[1]), bf16_unorder(hi[2]), bf16_unorder(hi[3]));
    }
  }
}

// The bounds of every block of the page table that reaches past start[b] (all of them without start), from the cache.
// One workgroup per block: its K rows are one contiguous run of tokens x HKV x D values, read 16 bytes a lane, a column
// of 8 (8-bit caches: 16) channels kept by as many lanes as the workgroup has to spare and joined through LDS. Minimum and
// maximum are taken on the bf16 bits as ordered 16-bit integers, two values an instruction; of an int8 cache in fp32, which
// holds code * scale exactly, and rounded outward once a lane. Bound by the K bytes: 145,592
// tokens of an FP8 cache (HKV 2, D 256, blocks of 32) 18.6 us, 84 MB at 4.5 TB/s; without minimum and maximum at all 4%
// less, with non-temporal loads 8% more, and 1.5 us more while lanes stored dwords 32 bytes apart. As an int8 cache the
// same tokens take 26.4 us, 84 MB at 3.2 TB/s: a convert, a product, a minimum and a maximum a value in fp32.
template <int T>
__global__ __launch_bounds__(256) void paged_key_bounds_kernel(
    const unsigned char* __restrict__ cache, const uint16_t* __restrict__ scales, uint16_t* __restrict__ bounds, const int* __restrict__ indptr,
    const int* __restrict__ indices, const int* __restrict__ last, const int* __restrict__ start, int nnz, int batch,
    int hkv, int d, int page_size, int block, int64_t num_pages, float inv_scale, int* __restrict__ status) {
  constexpr int N = T ? 8 : 4;      // dwords of bf16 pairs a lane keeps
  constexpr int E = 2 * N;           // channels a lane keeps
  constexpr int B = T ? 1 : 2;      // bytes of a stored value
  __shared__ __align__(16) axk_s16x2 s_lo[256 * N], s_hi[256 * N];
  const int tid = threadIdx.x;
  const int bpp = page_size / block;
  const int entry = blockIdx.x / bpp, sub = blockIdx.x - entry * bpp;
  const int page = indices[entry];
  const Owner own = owner_of(indptr, last, batch, page_size, nnz, entry);
  if (own.b >= batch) return;  // past the last sequence
  const Seq s = own.s;
  const int64_t t0 = (int64_t)(entry - s.pb) * page_size + (int64_t)sub * block;
  const int rows = (int)min((int64_t)block, s.len - t0);
  if (entry < s.pb || rows <= 0 || (start && t0 + block <= start[own.b])) return;
  if (page < 0 || page >= num_pages) {
    if (status && tid == 0) *status = 1;
    return;
  }
  const int row = hkv * d;
  const int cols = row / E;  // lanes that one token row takes
  const int64_t first = (int64_t)page * 2 * page_size + (int64_t)sub * block;  // the block's first K row
  const unsigned char* src = cache + first * row * B;
  uint16_t* dst = bounds + ((int64_t)page * bpp + sub) * hkv * 2 * d;
  for (int c0 = 0; c0 < cols; c0 += 256) {
    const int w = min(cols - c0, 256), lanes = 256 / w;  // columns of this pass, and lanes to each
    const int rl = tid / w, c = c0 + tid - rl * w;
    const uint16_t* sc = T == kI8 ? scales + first * hkv + (unsigned)(c * E) / (unsigned)d : nullptr;  // a lane's head
    axk_s16x2 lo[N], hi[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo[e] = (axk_s16x2)(short)0x7fff;
      hi[e] = (axk_s16x2)(short)-0x8000;
    }
    float lof[T == kI8 ? E : 1], hif[T == kI8 ? E : 1];  // int8 keys in fp32, where the product is exact; NaN stays
    if constexpr (T == kI8) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lof[e] = INFINITY;
        hif[e] = -INFINITY;
      }
    }
    if (rl < lanes) {
#pragma unroll 4
      for (int t = rl; t < rows; t += lanes) {
        const axk_u32x4 w4 = *reinterpret_cast<const axk_u32x4*>(src + ((int64_t)t * row + c * E) * B);
        if constexpr (T == kI8) {
          const float s = bf16_bits_to_f32(sc[(int64_t)t * hkv]);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float x = i8_code(w4[e / 4], e % 4) * s;
            lof[e] = __builtin_elementwise_minimum(lof[e], x);
            hif[e] = __builtin_elementwise_maximum(hif[e], x);
          }
        } else {
          uint32_t x[N];
          stored_pairs<T>(w4, inv_scale, x);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            lo[e] = __builtin_elementwise_min(lo[e], bf16_order(x[e]));
            hi[e] = __builtin_elementwise_max(hi[e], bf16_order(x[e]));
          }
        }
      }
    }
    if constexpr (T == kI8) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        lo[e] = bf16_order(high_halves(bf16_down(lof[2 * e]), bf16_down(lof[2 * e + 1])));
        hi[e] = bf16_order(high_halves(bf16_up(hif[2 * e]), bf16_up(hif[2 * e + 1])));
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e) {
      s_lo[tid * N + e] = lo[e];
      s_hi[tid * N + e] = hi[e];
    }
    __syncthreads();
    for (int i = tid; i < w * N; i += 256) {  // dword i of the pass's row: consecutive lanes store consecutive dwords
      axk_s16x2 l = s_lo[i], h = s_hi[i];
      for (int j = 1; j < lanes; ++j) {
        l = __builtin_elementwise_min(l, s_lo[j * w * N + i]);
        h = __builtin_elementwise_max(h, s_hi[j * w * N + i]);
      }
      const int at = c0 * E + 2 * i, head = (int)((unsigned)at / (unsigned)d);
      uint32_t* o = reinterpret_cast<uint32_t*>(dst + (int64_t)head * 2 * d + (at - head * d));
      o[0] = bf16_unorder(l);
      o[d / 2] = bf16_unorder(h);
    }
  }
}

// ---- block scores ----
// max(q lo, q hi) per channel is q+ hi + q- lo with q+ = max(q, 0), q- = min(q, 0): the score of 16 blocks for the 16
// (padded) heads of a group is one chain of 2 D / 32 16x16x32 MFMAs, blocks as rows, and a block's bounds are read once.
// One wave per (16 blocks, KV head); a tile that spans sequences is computed once with each one's queries. Bound by the
// bounds' bytes: 8 sequences of 131072 tokens in blocks of 64 (HKV 4, D 256) 16.5 us, 68 MB at 4.1 TB/s, all of its waves
// at once. With the rows through LDS as in the decode below the same took 18.2 us, since half as many waves fit (and one
// sequence of 5003 tokens 4.6 against 5.6).
//
// Where a bound is infinite, the product that the split leaves at zero is 0 inf = NaN, though max(q lo, q hi) is not. So a
// block whose sum came out NaN is summed again as the formula stands, head by head, after the others: a lane's block and
// channels as there, its bounds read again (kept, they would cost every wave registers: 160 instead of 92 at D 256).
template <int D>
AXK_DEV float plain_score(const uint16_t* __restrict__ q, const uint16_t* __restrict__ row, int group) {
  float best = -INFINITY;
#pragma unroll 1
  for (int head = 0; head < group; ++head) {
    float sum = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
      const axk_bf16x8 x = load_bf16x8(q + (int64_t)head * D + d), lo = load_bf16x8(row + d), hi = load_bf16x8(row + D + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += __builtin_elementwise_maximum((float)x[e] * (float)lo[e], (float)x[e] * (float)hi[e]);
    }
    best = __builtin_elementwise_maximum(best, xor32_sum(xor16_sum(sum)));
  }
  return best;
}

template <int D>
__global__ __launch_bounds__(256) void paged_block_scores_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ bounds, const int* __restrict__ indptr,
    const int* __restrict__ indices, const int* __restrict__ last, float* __restrict__ scores, int nnz, int batch,
    int hq, int hkv, int page_size, int block, int64_t num_pages, unsigned units, int* __restrict__ status) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const unsigned unit = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int group = hq / hkv, bpp = page_size / block;
  const int total = nnz * bpp;
  const int tile = (int)(unit / (unsigned)hkv);
  const int h = (int)(unit - (unsigned)tile * hkv);
  // lane l16 of each lane group looks at block tile * 16 + l16
  const int f = tile * 16 + l16;
  const int e = (int)((unsigned)min(f, total - 1) / (unsigned)bpp);
  const int id = indices[e];
  const int e0 = __builtin_amdgcn_readlane(e, 0), e1 = __builtin_amdgcn_readlane(e, 15);
  Owner own = owner_of(indptr, last, batch, page_size, nnz, e0);
  const bool good = id >= 0 && id < num_pages;
  const int sub = f - e * bpp;
  const uint16_t* row = bounds + (((int64_t)(good ? id : 0) * bpp + (f < total ? sub : 0)) * hkv + h) * 2 * D + 8 * g;
  axk_bf16x8 lo[D / 32], hi[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    lo[s] = load_bf16x8(row + 32 * s);
    hi[s] = load_bf16x8(row + D + 32 * s);
  }
  int again = 0;  // lane 16 g, bit i: the sum of block 4 g + i came out NaN
  for (int b = own.b; b < batch; ++b) {  // the sequences whose entries reach into the tile
    const Seq sq = b == own.b ? own.s : seq_of(indptr, last, b, page_size, nnz);
    if (sq.pb > e1) break;
    axk_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const uint16_t* qr = q + ((int64_t)b * hq + h * group + l16) * D + 8 * g;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      // bf16 sign and order agree with those of the bits as 16-bit integers
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const s16x8 x = l16 < group ? *reinterpret_cast<const s16x8*>(qr + 32 * s) : (s16x8)(short)0;
      const s16x8 pos = __builtin_elementwise_max(x, (s16x8)(short)0), neg = __builtin_elementwise_min(x, (s16x8)(short)0);
      acc = mfma_bf16_16x16x32(hi[s], __builtin_bit_cast(axk_bf16x8, pos), acc);
      acc = mfma_bf16_16x16x32(lo[s], __builtin_bit_cast(axk_bf16x8, neg), acc);
    }
    // acc[i]: block tile * 16 + 4 g + i, head l16: the maximum over the group's heads
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = l16 < group ? acc[i] : -INFINITY;
      float n = x != x ? x : 0.f;  // a NaN of any head is the block's score (fmaxf would drop it)
      x = fmaxf(x, dpp_move<0xB1>(x, x));
      x = fmaxf(x, dpp_move<0x4E>(x, x));
      x = fmaxf(x, dpp_move<0x141>(x, x));
      x = fmaxf(x, dpp_move<0x140>(x, x));
      n = group_sum<16>(n);
      if (n != n) x = n;
      const int fi = tile * 16 + 4 * g + i;
      const int64_t t0 = (int64_t)(fi - sq.pb * bpp) * block;  // the block's first token
      const bool bad = __shfl((int)!good, 4 * g + i, 64) != 0;
      if (l16 == 0 && fi < total && t0 >= 0 && t0 < (int64_t)sq.np * page_size) {
        const bool there = t0 < sq.len;
        scores[(int64_t)h * total + fi] = there && !bad ? x : -INFINITY;
        if (there && bad && status) *status = 1;
        if (there && !bad && x != x) again |= 1 << i;
      }
    }
  }
  if (!__any(again)) return;
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");  // the NaNs are stored before what replaces them
  again = __shfl(again, 16 * (l16 >> 2), 64) >> (l16 & 3) & 1;  // of this lane's block
  for (int b = own.b; b < batch; ++b) {
    const Seq sq = seq_of(indptr, last, b, page_size, nnz);
    if (sq.pb > e1) break;
    const float x = plain_score<D>(q + ((int64_t)b * hq + h * group) * D + 8 * g, row, group);
    const int64_t t0 = (int64_t)(f - sq.pb * bpp) * block;
    if (g == 0 && again && t0 >= 0 && t0 < sq.len) scores[(int64_t)h * total + f] = x;
  }
}

// ---- the `want` largest of a row ----
// Radix selection by one workgroup of T threads, K consecutive keys each in registers (a longer row is read again, T K keys
// at a time, in each step). Keys are taken relative to the row's smallest, and log2(4 T) bits at a time, from the highest
// that the row's range has, are counted in 4 T bins of LDS, until the smallest key that is taken is known or all keys that
// agree with it so far are taken: two rounds as a rule. 256 of 8192 scores for 32 rows 9.7 us, 64 of 313 4.0: latency, as
// the bytes take 0.2 us; how it divides between loads, counts, scans and barriers has not been measured for this form.
// (With 256 bins of the raw bits the former took 19.6: most scores share sign and exponent, and adds to one address wait
// for each other.) Equal keys at the border are taken by the lowest index. load(at, n, key) fetches a thread's n keys from
// index `at`; emit(i, taken, rank) is called for every index, rank = the indices below i that are taken; done(base, n, k)
// after the n indices of a tile, k of them taken.
template <class Key, int T>
struct PickLds {
  unsigned hist[4 * T];
  Key lo[T / 64], hi[T / 64];
  unsigned sums[T / 64];
  unsigned digit, above, inside;
};

// A 32- or 64-bit value moved by DPP (lanes without a source keep theirs), and a wave's minimum and maximum of it.
template <int CTRL, int ROW_MASK = 0xF>
AXK_DEV uint32_t dpp_key(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, ROW_MASK, 0xF, false);
}
template <int CTRL, int ROW_MASK = 0xF>
AXK_DEV uint64_t dpp_key(uint64_t v) {
  return (uint64_t)dpp_key<CTRL, ROW_MASK>((uint32_t)(v >> 32)) << 32 | dpp_key<CTRL, ROW_MASK>((uint32_t)v);
}
AXK_DEV uint32_t lane63_key(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
AXK_DEV uint64_t lane63_key(uint64_t v) { return (uint64_t)lane63_key((uint32_t)(v >> 32)) << 32 | lane63_key((uint32_t)v); }
template <class Key, class Op>
AXK_DEV Key wave_key(Key v, const Op& op) {
  v = op(v, dpp_key<0xB1>(v));
  v = op(v, dpp_key<0x4E>(v));
  v = op(v, dpp_key<0x141>(v));
  v = op(v, dpp_key<0x140>(v));
  v = op(v, dpp_key<0x142, 0xA>(v));
  v = op(v, dpp_key<0x143, 0xC>(v));
  return lane63_key(v);
}

template <class Key, int T, int K, class Load, class Emit, class Done>
AXK_DEV void pick_largest(int count, int want, const Load& load, const Emit& emit, const Done& done, PickLds<Key, T>& lds) {
  constexpr int kTile = T * K, kBits = 8 * sizeof(Key), kStep = T == 1024 ? 12 : 10;
  static_assert(4 * T == 1 << kStep, "four bins a thread");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = (count + kTile - 1) / kTile;
  const int per = tiles > 1 ? K : (count + T - 1) / T;  // consecutive indices a thread holds
  Key key[K];
  int mine = 0;  // how many of them there are
  auto load_tile = [&](int t) {
    mine = min(max(count - t * kTile - tid * per, 0), per);
    load(t * kTile + tid * per, mine, key);
  };
  if (tiles == 1) load_tile(0);
  *reinterpret_cast<uint4*>(&lds.hist[4 * tid]) = make_uint4(0, 0, 0, 0);
  Key lo = ~(Key)0, hi = 0;
  for (int t = 0; t < tiles; ++t) {
    if (tiles > 1) load_tile(t);
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < mine) {
        lo = min(lo, key[i]);
        hi = max(hi, key[i]);
      }
  }
  lo = wave_key(lo, [](Key x, Key y) { return min(x, y); });
  hi = wave_key(hi, [](Key x, Key y) { return max(x, y); });
  if (lane == 0) {
    lds.lo[wave] = lo;
    lds.hi[wave] = hi;
  }
  __syncthreads();
  lo = lds.lo[lane % (T / 64)];
  hi = lds.hi[lane % (T / 64)];
  lo = wave_key(lo, [](Key x, Key y) { return min(x, y); });
  hi = wave_key(hi, [](Key x, Key y) { return max(x, y); });
  const Key range = hi - lo;
  int pos = range ? kBits - (sizeof(Key) == 8 ? __clzll((long long)range) : __clz((int)range)) : 0;  // bits of key - lo
  Key prefix = 0;                       // the border key's bits from `pos` up
  unsigned remaining = (unsigned)want;  // keys to take among those that agree with it
  bool all = false;
  while (pos > 0 && !all) {
    const int w = min(kStep, pos), from = pos;
    pos -= w;
    for (int t = 0; t < tiles; ++t) {
      if (tiles > 1) load_tile(t);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const Key x = key[i] - lo;
        if (i < mine && (from == kBits || (x ^ prefix) >> from == 0))
          atomicAdd(&lds.hist[(unsigned)(x >> pos) & ((1u << w) - 1u)], 1u);
      }
    }
    __syncthreads();
    // thread t: bins 4 (T - 1 - t) .. + 3, so that the scan runs from the top
    uint4* bins = reinterpret_cast<uint4*>(&lds.hist[4 * (T - 1 - tid)]);
    const uint4 c4 = *bins;
    *bins = make_uint4(0, 0, 0, 0);
    const unsigned c[4] = {c4.w, c4.z, c4.y, c4.x}, sum = c[0] + c[1] + c[2] + c[3];
    const unsigned incl = wave_scan(sum);
    if (lane == 63) lds.sums[wave] = incl;
    __syncthreads();
    unsigned before = incl - sum;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) before += i < wave ? lds.sums[i] : 0u;
    if (before < remaining && remaining <= before + sum) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < remaining && remaining <= before + c[i]) {
          lds.digit = 4 * (T - 1 - tid) + 3 - i;
          lds.above = before;
          lds.inside = c[i];
        }
        before += c[i];
      }
    }
    __syncthreads();
    prefix |= (Key)lds.digit << pos;
    remaining -= lds.above;
    all = lds.inside == remaining;
  }
  // taken: keys above the border (compared from `pos` up), and the first `remaining` of those on it
  const Key border = prefix >> pos;
  unsigned above0 = 0, on0 = 0;
  for (int t = 0; t < tiles; ++t) {
    if (tiles > 1) load_tile(t);
    unsigned up = 0, eq = 0;  // a bit a key: above the border, on it
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < mine) {
        const Key x = (key[i] - lo) >> pos;
        up |= (x > border ? 1u : 0u) << i;
        eq |= (x == border ? 1u : 0u) << i;
      }
    // above in the high half, on the border in the low half: at most T K < 65536 of each
    const unsigned n = ((unsigned)__popc(up) << 16) + (unsigned)__popc(eq), incl = wave_scan(n);
    __syncthreads();  // the sums of the tile before have been read
    if (lane == 63) lds.sums[wave] = incl;
    __syncthreads();
    unsigned before = incl - n, total = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) {
      const unsigned x = lds.sums[i];
      before += i < wave ? x : 0u;
      total += x;
    }
    unsigned above = above0 + (before >> 16), on = on0 + (before & 0xffffu);
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      const unsigned u = (up >> i) & 1u, q = (eq >> i) & 1u;
      emit(t * kTile + tid * per + i, u || (q && on < remaining), (int)(above + min(on, remaining)));
      above += u;
      on += q;
    }
    const unsigned before_tile = above0 + min(on0, remaining);
    above0 += total >> 16;
    on0 += total & 0xffffu;
    done(t * kTile, min(count - t * kTile, kTile), (int)(above0 + min(on0, remaining) - before_tile));
  }
}

// n <= K floats from p, four at a time where all K are there (p need not be 16-byte aligned)
template <int K>
AXK_DEV void load_run(const float* __restrict__ p, int n, float (&x)[K]) {
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  if (K % 4 == 0 && n == K) {
#pragma unroll
    for (int i = 0; i < K; i += 4) {
      const f4 v = *reinterpret_cast<const f4*>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i + j] = v[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < K; ++i) x[i] = i < n ? p[i] : 0.f;
  }
}

// Floats as integers of the same order: NaN of either sign above +inf, zeros of either sign equal.
AXK_DEV uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  if (x != x) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
AXK_DEV uint64_t order_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  if (x != x) return ~0ull;
  return u >> 63 ? ~u : u | (1ull << 63);
}

// One workgroup per (sequence, KV head): its n best blocks, the first `first` and last `keep_last` always among them.
template <int T, int K>
AXK_DEV void select_row(const float* __restrict__ row, int count, int want, int* __restrict__ out, int first,
                        PickLds<uint32_t, T>& lds) {
  pick_largest<uint32_t, T, K>(
      count, want,
      [&](int at, int n, uint32_t(&key)[K]) {
        float x[K];
        load_run<K>(row + at, n, x);
#pragma unroll
        for (int i = 0; i < K; ++i) key[i] = order_key(x[i]);
      },
      [&](int i, bool taken, int rank) {
        if (taken) out[rank] = first + i;
      },
      [](int, int, int) {}, lds);
}
template <int T>
__global__ __launch_bounds__(T) void paged_select_blocks_kernel(const float* __restrict__ scores,
                                                                const int* __restrict__ indptr,
                                                                const int* __restrict__ last, int* __restrict__ out,
                                                                int nnz, int hkv, int page_size, int block, int n,
                                                                int first, int keep_last) {
  __shared__ PickLds<uint32_t, T> lds;
  const int tid = threadIdx.x, b = blockIdx.x / hkv, h = blockIdx.x - b * hkv;
  const Seq s = seq_of(indptr, last, b, page_size, nnz);
  const int bpp = page_size / block;
  const int nb = blocks_of(s, block);
  int* o = out + (int64_t)blockIdx.x * n;
  if (nb <= n) {
    for (int i = tid; i < n; i += T) o[i] = i < nb ? i : -1;
    return;
  }
  for (int i = tid; i < first; i += T) o[i] = i;
  for (int i = tid; i < keep_last; i += T) o[n - keep_last + i] = nb - keep_last + i;
  const int want = n - first - keep_last, count = nb - first - keep_last;
  if (want == 0) return;
  const float* row = scores + (int64_t)h * nnz * bpp + (int64_t)s.pb * bpp + first;
  if (count <= 2 * T) select_row<T, 2>(row, count, want, o + first, first, lds);
  else if (count <= 8 * T || T < 1024) select_row<T, 8>(row, count, want, o + first, first, lds);
  else select_row<T, 16>(row, count, want, o + first, first, lds);
}

// ---- decode over blocks ----
// One query token per sequence over the listed blocks of each KV head (or all of them), split over pieces of `ps`
// subtiles of 16 tokens. Everything a wave needs stays in its registers; it takes two subtiles (32 tokens) a step:
//   S^T = K Q^T   16x16x32 MFMA, K rows through LDS as the A operand (lane = token, 16 bytes of its row), Q the B operand,
//                 the group's heads as columns;
//   softmax       running maximum and sum per head, fp32, exp2 domain;
//   O^T += V^T P^T  the score accumulator is the P^T operand as it stands if MFMA k index (lane group g, j) is token
//                 4 g + j % 4 of subtile j / 4. V rows are loaded in that order, lane l16 holding D / 16 channels of eight
//                 tokens, so that the transposition V^T needs is one byte permute per two values, without LDS.
// The four waves of a piece take its steps in turn and are joined through LDS; pieces by the merge kernel.
// Bound by HBM: 64 blocks of 64 for 8 sequences of 131072 tokens (HQ 32, HKV 4, D 256) 28.2 us, 134 MB at 4.8 TB/s; all
// 145,592 tokens of 16 sequences (HQ 16, HKV 2) of an FP8 cache 29.9 us, 149 MB at 5.0 TB/s, of an int8 cache 32.9 us, 151 MB
// at 4.6; of these some 5 us are the chain of lookups before the first load (list, page, rows) and the join after the last.
// (The decode over whole bf16 caches in paged_attn.hip reads 6.1 TB/s.) As many pieces as run at once are best: with three
// quarters of them the former took 17% longer, with half as many again 3%, and the latter 25%.
template <int D, int T>
struct BlkCfg {
  static constexpr int B = T ? 1 : 2;              // bytes of a stored value
  static constexpr int RB = D * B;                 // bytes of a token's row of one head
  static constexpr int CR = RB / 16;               // ... in 16-byte chunks
  static constexpr int KI = 32 * RB / 1024;        // direct-to-LDS loads (64 lanes x 16 bytes) of a step's K
  static constexpr int KL = RB / 64;               // 16-byte K fragments a lane reads per subtile
  static constexpr int KS = D / 32;                // QK k-steps
  static constexpr int E = T ? D / 16 : (D >= 128 ? 8 : D / 16);  // channels of a V load
  static constexpr int NH = D / 16 / E;            // V loads a lane makes per token
  static constexpr int VW = E * B / 4;             // dwords of a V load
  static constexpr int ACC = D / 16;               // 16x16 O^T tiles
  static constexpr int Q = ACC / 4;                // ... that a wave gives out at the end
  static constexpr int KT = 32 * RB;               // bytes of a step's K in LDS, one buffer a wave
  static constexpr int LDS = 4 * KT > 12 * Q * 1024 ? 4 * KT : 12 * Q * 1024;  // the join at the end reuses them
  // Chunk c of row r lies at chunk c ^ swz(r) of its row in LDS: the 16 rows that lanes read one chunk of then fall on 16
  // different 16-byte columns of the 256 bytes that LDS gives at a time.
  static AXK_DEV int swz(int r) { return CR >= 16 ? r & 15 : r / (16 / (CR < 16 ? CR : 16)) & (CR - 1); }
};

struct BlkArgs {
  const uint16_t* q;
  const unsigned char* cache;
  const uint16_t* kv_scales;  // of an int8 cache
  const int *indptr, *indices, *last;
  const int* blocks;  // [batch, hkv, n], or null: every block
  int n, block;
  int nnz, batch, hq, hkv, page;
  int64_t num_pages;
  float scale;      // sm_scale * log2(e)
  float inv_scale;  // of an FP8 cache
  int ps;           // subtiles of a piece
  int pieces;       // pieces of a row (listed blocks), or of all sequences of one KV head (every block)
  int direct;       // every row is one piece: no merge
  uint16_t* out;
  float2* ml;       // [rows or hkv][pieces][group]: maximum and sum
  float* po;        // ... [D]
  float2* stat;     // per (row or hkv, subtile, head) reference and sum, for the page weights; null: not wanted
  int* status;
};

// Which sequence and which of its pieces flat piece `it` of a KV head is, where every block is attended: the pieces of
// a sequence are as many as its subtiles need. b = batch past the last one.
struct PieceOf {
  int b, piece;
  Seq s;
};
// (One at least where it has pages, so that pages without a token get their weights too.)
AXK_DEV int pieces_of(const Seq& s, int ps) { return s.np ? max((int)((unsigned)(subs_of(s) + ps - 1) / (unsigned)ps), 1) : 0; }
AXK_DEV PieceOf find_piece(const BlkArgs& a, int it) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 256) {  // 256 sequences a round trip to memory, each wave for itself
    int lo[4], hi[4], last[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = min(b0 + 64 * i + lane, a.batch - 1);
      lo[i] = a.indptr[b];
      hi[i] = a.indptr[b + 1];
      last[i] = a.last[b];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (b0 + 64 * i >= a.batch) break;
      const int n = b0 + 64 * i + lane < a.batch ? pieces_of(seq_from(lo[i], hi[i], last[i], a.page, a.nnz), a.ps) : 0;
      const int before = base + (int)wave_scan((unsigned)n) - n;
      // (offsets of indptr that fall back can make the sums pass 32 bits: such pieces are nobody's)
      const uint64_t mine = __ballot(before >= 0 && it >= before && it - before < n);
      if (mine) {
        const int src = __ffsll((unsigned long long)mine) - 1;
        return {b0 + 64 * i + src, it - __builtin_amdgcn_readlane(before, src),
                seq_from(__builtin_amdgcn_readlane(lo[i], src), __builtin_amdgcn_readlane(hi[i], src),
                         __builtin_amdgcn_readlane(last[i], src), a.page, a.nnz)};
      }
      base = __builtin_amdgcn_readlane(before + n, 63);
    }
  }
  return {a.batch, 0, {0, 0, 0}};
}
// Pieces of the sequences before b, where every block is attended (each wave for itself).
AXK_DEV int pieces_before(const BlkArgs& a, int b) {
  int n = 0;
  for (int i = threadIdx.x & 63; i < b; i += 64) n += pieces_of(seq_of(a.indptr, a.last, i, a.page, a.nnz), a.ps);
  return wave_total(n);
}

// Whether a listed block is neither padding (-1) nor a block of the sequence that lies above its predecessor in the list,
// which is no padding either (prev: kNoPrev for the first).
constexpr int kNoPrev = -2;
AXK_DEV bool bad_block(int id, int prev, int nblocks) {
  return id < -1 || id >= nblocks || (id >= 0 && (prev >= id || prev == -1));
}

// A wave-uniform 64-bit value in scalar registers.
AXK_DEV int64_t uniform_i64(int64_t x) {
  return (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

constexpr int kMaxPs = 128;  // subtiles of a piece, at most (two a lane)

template <int D, int T>
__global__ __launch_bounds__(256, 2) void paged_blocks_kernel(const BlkArgs a) {
  using C = BlkCfg<D, T>;
  constexpr int Q = C::Q;
  extern __shared__ __align__(1024) unsigned char s_k[];  // C::LDS bytes
  __shared__ int64_t s_row[kMaxPs];
  __shared__ int s_valid[kMaxPs];
  __shared__ float s_m[4][16], s_l[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
  const int group = a.hq / a.hkv;
  int b, h, piece;
  int64_t item;
  Seq s;
  const int spb = a.block / kSub;
  int id = -1, prev = kNoPrev;  // thread i: the listed block that subtile i of the piece lies in, and the one before it
  if (a.blocks) {
    item = blockIdx.x;
    const int row = blockIdx.x / a.pieces;
    piece = blockIdx.x - row * a.pieces;
    b = row / a.hkv;
    h = row - b * a.hkv;
    const int slot = (int)((unsigned)(piece * a.ps + tid) / (unsigned)spb);
    if (tid < a.ps && slot < a.n) {
      const int* list = a.blocks + (int64_t)row * a.n + slot;
      id = list[0];
      if (slot) prev = list[-1];
    }
    s = seq_of(a.indptr, a.last, b, a.page, a.nnz);
  } else {
    h = blockIdx.y;
    item = (int64_t)h * a.pieces + blockIdx.x;
    const PieceOf p = find_piece(a, blockIdx.x);
    b = p.b;
    piece = p.piece;
    s = p.s;
    if (b >= a.batch) return;
  }
  // Q first: its loads are under way while the subtiles' places are looked up
  axk_bf16x8 qf[C::KS];
#pragma unroll
  for (int i = 0; i < C::KS; ++i) {
    const int at = T ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
    qf[i] = l16 < group ? load_bf16x8(a.q + ((int64_t)b * a.hq + h * group + l16) * D + at) : zero_bf16x8();
  }
  // the piece's subtiles: where each lies in the cache, and how many of its tokens count
  const int64_t rowb = (int64_t)a.hkv * D * C::B;  // bytes of a token row
  const int spp = a.page / kSub;
  const int nsub = a.blocks ? a.n * spb : subs_of(s);  // of the row
  const int sub0 = piece * a.ps;
  const int count = min(a.ps, nsub - sub0);
  if (tid < a.ps) {
    int valid = 0;
    int64_t base = 0;
    if (tid < count) {
      int at = sub0 + tid;  // the subtile's place in the sequence
      bool bad = false;
      if (a.blocks) {
        bad = bad_block(id, prev, blocks_of(s, a.block));
        at = bad || id < 0 ? subs_of(s) : id * spb + (int)((unsigned)at % (unsigned)spb);
      }
      valid = (int)min(max(s.len - (int64_t)at * kSub, (int64_t)0), (int64_t)kSub);
      if (valid) {
        const int p = (int)((unsigned)at / (unsigned)spp), page = a.indices[s.pb + p];
        if (page < 0 || page >= a.num_pages) {
          bad = true;
          valid = 0;
        } else {
          base = (int64_t)page * 2 * a.page + (at - p * spp) * kSub;
        }
      }
      if (bad && a.status) *a.status = 1;
    }
    s_row[tid] = base;
    s_valid[tid] = valid;
  }
  __syncthreads();
  // one past the last subtile with a token: what follows is padding of the list
  const uint64_t low = __ballot(lane < a.ps && s_valid[lane] > 0), high = __ballot(64 + lane < a.ps && s_valid[min(64 + lane, a.ps - 1)] > 0);
  const int end = high ? 128 - __clzll((long long)high) : low ? 64 - __clzll((long long)low) : 0;
  const int64_t stat_at = (a.blocks ? ((int64_t)b * a.hkv + h) * nsub : ((int64_t)h * a.nnz + s.pb) * spp) + sub0;
  if (a.stat)
    for (int i = ((end + 1) & ~1) * group + tid; i < count * group; i += 256)
      a.stat[stat_at * group + i] = make_float2(0.f, 0.f);

  axk_f32x4 acc[C::ACC];
#pragma unroll
  for (int i = 0; i < C::ACC; ++i) acc[i] = (axk_f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const unsigned char* cache_h = a.cache + (int64_t)h * D * C::B;
  const uint32_t v_off = (uint32_t)(4 * g * rowb + l16 * C::E * C::B);
  typedef uint32_t vload __attribute__((ext_vector_type(C::VW)));
  // K of step t to this wave's buffer, whole rows an instruction (a fragment's 64 bytes of 16 rows, straight to registers,
  // ask the L2 for every line twice). Nothing else touches the buffer, so no barrier is needed.
  unsigned char* kbuf = s_k + wave * C::KT;
  constexpr int kRows = 1024 / C::RB;  // rows of one load
  auto load_k = [&](int t) {
    const unsigned char* sub[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) sub[u] = cache_h + uniform_i64(s_row[2 * t + u]) * rowb;
#pragma unroll
    for (int i = 0; i < C::KI; ++i) {
      const int r = (i * kRows + lane / C::CR) % kSub;  // of its subtile
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(sub[i * kRows / kSub] + (uint32_t)(r * rowb + ((lane % C::CR) ^ C::swz(r)) * 16)),
          (__attribute__((address_space(3))) void*)(kbuf + i * 1024), 16, 0, 2);
    }
  };
  const uint32_t k_at = (uint32_t)(l16 * C::RB + ((g ^ C::swz(l16)) * 16));  // chunk g of row l16; chunk 4 i + g: ^ 64 i
  const int tiles = (end + 1) / 2;
  if (wave < tiles) load_k(wave);
  for (int t = wave; t < tiles; t += 4) {
    const int nv0 = __builtin_amdgcn_readfirstlane(s_valid[2 * t]), nv1 = __builtin_amdgcn_readfirstlane(s_valid[2 * t + 1]);
    vload vr[8][C::NH];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const unsigned char* p = cache_h + (uniform_i64(s_row[2 * t + u]) + a.page) * rowb;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < C::NH; ++n)
          vr[4 * u + j][n] = __builtin_nontemporal_load(
              reinterpret_cast<const vload*>(p + v_off + j * (uint32_t)rowb + n * 16 * C::E * C::B));
    }
    // int8: lane (plane, subtile, token) loads one scale, zero where the token does not count
    float ks[8], vs[8], own = 0.f;
    if constexpr (T == kI8) {
      const int u = g & 1, plane = g >> 1;
      if (l16 < (u ? nv1 : nv0))
        own = bf16_bits_to_f32(a.kv_scales[(s_row[2 * t + u] + plane * a.page + l16) * a.hkv + h]);
    }
    // This step's K has landed in LDS (the compiler waits for registers only), and its V with it. (The other waves' loads keep
    // the memory busy meanwhile; a wait for K alone has not been measured.)
    wait_vmcnt<0>();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (T == kI8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // the scales of this lane's tokens: 4 g + j % 4 of subtile j / 4
        ks[j] = __shfl(own, (j >> 2) * 16 + 4 * g + (j & 3), 64);
        vs[j] = __shfl(own, 32 + (j >> 2) * 16 + 4 * g + (j & 3), 64);
      }
    }
    axk_f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = (axk_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < C::KL; ++i) {
        uint32_t x[T ? 8 : 4];
        stored_pairs<T>(*reinterpret_cast<const axk_u32x4*>(kbuf + u * kSub * C::RB + (k_at ^ (64 * i))), a.inv_scale, x);
        const axk_u32x4 x0 = {x[0], x[1], x[2], x[3]};
        sc[u] = mfma_bf16_16x16x32(__builtin_bit_cast(axk_bf16x8, x0), qf[T ? 2 * i : i], sc[u]);
        if constexpr (T != kBf16) {
          const axk_u32x4 x1 = {x[4], x[5], x[6], x[7]};
          sc[u] = mfma_bf16_16x16x32(__builtin_bit_cast(axk_bf16x8, x1), qf[2 * i + 1], sc[u]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t + 4 < tiles) load_k(t + 4);
    __builtin_amdgcn_sched_barrier(0);
    // sc[u][i]: token 4 g + i of subtile u, head l16
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T == kI8) {
        sc[0][i] *= ks[i];
        sc[1][i] *= ks[4 + i];
      }
      x[i] = 4 * g + i < nv0 ? sc[0][i] * a.scale : -INFINITY;
      x[4 + i] = 4 * g + i < nv1 ? sc[1][i] * a.scale : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    top = fmaxf(m, xor32_max(xor16_max(top)));
    const float ref = top == -INFINITY ? 0.f : top;  // nothing counted yet: exp2(-inf) = 0 throughout
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] - ref);
    const float sum0 = (x[0] + x[1]) + (x[2] + x[3]), sum1 = (x[4] + x[5]) + (x[6] + x[7]);
    l = l * alpha + (sum0 + sum1);
    if (a.stat) {
      const float t0 = xor32_sum(xor16_sum(sum0)), t1 = xor32_sum(xor16_sum(sum1));
      if (g < 2 && 2 * t + g < count && l16 < group)  // lane group 0: the first subtile, 1: the second
        a.stat[(stat_at + 2 * t + g) * group + l16] = make_float2(ref, g ? t1 : t0);
    }
    if (__any(alpha != 1.0f)) {
#pragma unroll
      for (int i = 0; i < C::ACC; ++i) acc[i] *= alpha;
    }
    if constexpr (T == kI8) {  // V's scales go with the probabilities
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= vs[i];
    }
    // Probabilities meet V in bf16, as V itself is held (half a step, 2^-8 of each, which averages out over the tokens:
    // outputs are off by 1.7e-3 of their size, those of fp32 probabilities by as much, their own rounding). l keeps fp32.
    const axk_u32x4 pw = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                          pack_bf16x2(x[6], x[7])};
    const axk_bf16x8 pf = __builtin_bit_cast(axk_bf16x8, pw);
    if (nv0 < kSub || nv1 < kSub) {  // rows that do not count may hold anything: 0 * NaN is not 0
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (4 * g + (j & 3) >= (j < 4 ? nv0 : nv1))
#pragma unroll
          for (int n = 0; n < C::NH; ++n) vr[j][n] = (vload)0u;
    }
#pragma unroll
    for (int n = 0; n < C::NH; ++n)
#pragma unroll
      for (int w = 0; w < C::VW; ++w) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (T != kBf16) {
          uint32_t lo[4], hi[4];  // bytes (c, c + 1) of token pairs: [t.c, t'.c, t.c+1, t'.c+1]
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            lo[p] = __builtin_amdgcn_perm(vr[2 * p + 1][n][w], vr[2 * p][n][w], 0x05010400u);
            hi[p] = __builtin_amdgcn_perm(vr[2 * p + 1][n][w], vr[2 * p][n][w], 0x07030602u);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            axk_u32x4 f;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              f[p] = pair_of<T>(e < 2 ? lo[p] : hi[p], e & 1, a.inv_scale);
            }
            axk_f32x4& o = acc[n * C::E + 4 * w + e];
            o = mfma_bf16_16x16x32(__builtin_bit_cast(axk_bf16x8, f), pf, o);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            axk_u32x4 f;
#pragma unroll
            for (int p = 0; p < 4; ++p)
              f[p] = __builtin_amdgcn_perm(vr[2 * p + 1][n][w], vr[2 * p][n][w], e ? 0x07060302u : 0x05040100u);
            axk_f32x4& o = acc[n * C::E + 2 * w + e];
            o = mfma_bf16_16x16x32(__builtin_bit_cast(axk_bf16x8, f), pf, o);
          }
        }
      }
  }

  // the four waves' results against one maximum
  l = xor32_sum(xor16_sum(l));
  if (g == 0) {
    s_m[wave][l16] = m;
    s_l[wave][l16] = l;
  }
  __syncthreads();
  float top = fmaxf(fmaxf(s_m[0][l16], s_m[1][l16]), fmaxf(s_m[2][l16], s_m[3][l16]));
  if (top == -INFINITY) top = 0.f;
  const float mine = __builtin_amdgcn_exp2f(m - top);
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) l += s_l[w][l16] * __builtin_amdgcn_exp2f(s_m[w][l16] - top);
#pragma unroll
  for (int i = 0; i < C::ACC; ++i) acc[i] *= mine;
  // each wave gives out the sum of a quarter of the accumulators, and leaves the others theirs
  axk_f32x4* s_o = reinterpret_cast<axk_f32x4*>(s_k);
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (w != wave) {
#pragma unroll
      for (int i = 0; i < Q; ++i)
        s_o[((w * 3 + (wave < w ? wave : wave - 1)) * Q + i) * 64 + lane] = acc[w * Q + i];
    }
  __syncthreads();
  if (l16 >= group) return;
  const float inv = !a.direct ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
  if (!a.direct && wave == 0 && g == 0) a.ml[item * group + l16] = make_float2(top, l);
  uint16_t* out = a.out + ((int64_t)b * a.hq + h * group + l16) * D;
  float* po = a.po + (item * group + l16) * D;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    if (w == wave) {
      // lane: head l16, channels n 16 E + E (4 g + i) + e from acc[n E + e][i]
      axk_f32x4 o[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        o[i] = acc[w * Q + i];
#pragma unroll
        for (int j = 0; j < 3; ++j) o[i] += s_o[((w * 3 + j) * Q + i) * 64 + lane];
        o[i] *= inv;
      }
      const int at = w * Q / C::E * 16 * C::E + w * Q % C::E;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = at + C::E * (4 * g + i);
        if (a.direct) {
          if constexpr (Q == 1) {
            out[d] = (uint16_t)f32_to_bf16_bits(o[0][i]);
          } else {
#pragma unroll
            for (int e = 0; e < Q; e += 2) *reinterpret_cast<uint32_t*>(out + d + e) = pack_bf16x2(o[e][i], o[e + 1][i]);
          }
        } else {
          typedef float fq __attribute__((ext_vector_type(Q)));
          fq x;
#pragma unroll
          for (int e = 0; e < Q; ++e) x[e] = o[e][i];
          *reinterpret_cast<fq*>(po + d) = x;
        }
      }
    }
}

struct WeightArgs {
  const float* in;  // [hkv, nnz], null: zeros
  float* out;       // ..., null: not wanted
  float decay;
  int split;        // workgroups that share a row's output
};

// Two partial softmax sums as one; a sum of zero means that nothing was counted, whatever its maximum.
AXK_DEV float2 join(float2 x, float2 y) {
  if (y.y == 0.f) return x;
  if (x.y == 0.f) return y;
  const float top = fmaxf(x.x, y.x);
  return make_float2(top, x.y * __builtin_amdgcn_exp2f(x.x - top) + y.y * __builtin_amdgcn_exp2f(y.x - top));
}

AXK_DEV float2 join_pairs(uint2 m, uint2 l) {
  return join(make_float2(__uint_as_float(m.x), __uint_as_float(l.x)), make_float2(__uint_as_float(m.y), __uint_as_float(l.y)));
}

// A row's pieces: where they begin, how many the grid held (all of them, unless offsets of indptr overlap).
struct Pieces {
  int64_t item;
  int n;
};
// Joins the sums of head l16 over the row's pieces (`t`: that of piece tid / 16, already loaded), a part a wave in s_part.
AXK_DEV void join_pieces(float2 t, const float2* __restrict__ ml, int pieces, int group, float2 (*s_part)[16]) {
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  if (l16 < group)
    for (int p = (threadIdx.x >> 4) + 16; p < pieces; p += 16) t = join(t, ml[(int64_t)p * group + l16]);
  t = join_pairs(row_pair16(t.x), row_pair16(t.y));
  t = join_pairs(half_pair32(t.x), half_pair32(t.y));
  if (lane < 16) s_part[threadIdx.x >> 6][lane] = t;
  __syncthreads();
}

// A row's output, workgroup `part`: 64 float4s of its group x D values, a quarter of the pieces a wave. The first pieces'
// partial outputs are on their way while the sums are joined.
template <int D>
AXK_DEV void merge_output(const BlkArgs& a, int b, int h, int part, Pieces pc, float2 (*s_part)[16], axk_f32x4 (*s_o)[64]) {
  constexpr int kFirst = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = tid & 15, group = a.hq / a.hkv;
  const int per = group * D / 4, i = part * 64 + lane, head = min(i, per - 1) / (D / 4);
  const float2* ml = a.ml + pc.item * group;
  const axk_f32x4* po = reinterpret_cast<const axk_f32x4*>(a.po + (pc.n ? pc.item : 0) * group * D) + min(i, per - 1);
  const float2 none = make_float2(0.f, 0.f);
  float2 t = l16 < group && (tid >> 4) < pc.n ? ml[(tid >> 4) * group + l16] : none;
  axk_f32x4 v[kFirst];
  float2 x[kFirst];
#pragma unroll
  for (int k = 0; k < kFirst; ++k) {
    const int p = wave + 4 * k;
    x[k] = p < pc.n ? ml[(int64_t)p * group + head] : none;
    v[k] = po[(int64_t)max(min(p, pc.n - 1), 0) * per];  // past the end: not counted
  }
  join_pieces(t, ml, pc.n, group, s_part);
  t = join(join(s_part[0][head], s_part[1][head]), join(s_part[2][head], s_part[3][head]));
  const axk_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  axk_f32x4 o = zero;
#pragma unroll
  for (int k = 0; k < kFirst; ++k) {
    const axk_f32x4 y = __builtin_amdgcn_exp2f(x[k].x - t.x) * v[k];
    o += x[k].y == 0.f ? zero : y;  // a selection: what was not counted may be anything, and 0 * NaN is not 0
  }
#pragma unroll 8
  for (int p = wave + 4 * kFirst; p < pc.n; p += 4) {
    const float2 y = ml[(int64_t)p * group + head];
    const axk_f32x4 z = __builtin_amdgcn_exp2f(y.x - t.x) * po[(int64_t)p * per];
    o += y.y == 0.f ? zero : z;
  }
  s_o[wave][lane] = o;
  __syncthreads();
  if (wave == 0 && i < per) {
    o = ((s_o[0][lane] + s_o[1][lane]) + (s_o[2][lane] + s_o[3][lane])) * (t.y == 0.f ? 0.f : 1.0f / t.y);
    *reinterpret_cast<uint2*>(a.out + ((int64_t)b * a.hq + h * group) * D + 4 * i) =
        make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
  }
}

// The page weights of a row (listed blocks), or of the pages that begin in piece `piece` (every block): each subtile's sum
// against the row's joined maximum and sum. What is added up are units of subtiles (listed blocks, or pages), 64 at a time,
// four to 16 lanes, a head a lane, four subtiles of each together; the first ones are on their way while the sums are joined.
constexpr int kListLds = 2048;  // listed blocks whose shares are kept in LDS at a time
template <bool LISTED>
AXK_DEV void merge_weights(const BlkArgs& a, const WeightArgs& w, int b, int h, int piece, const Seq& s, Pieces pc,
                           float2 (*s_part)[16], float* s_share, int* s_page) {
  constexpr int NQ = LISTED ? 4 : 1;
  const int tid = threadIdx.x, l16 = tid & 15, r16 = tid >> 4, group = a.hq / a.hkv;
  const float2* ml = a.ml + pc.item * group;
  const float2 none = make_float2(0.f, 0.f);
  float2 t = l16 < group && r16 < pc.n ? ml[r16 * group + l16] : none;
  const int spp = a.page / kSub, spb = a.block / kSub, bpp = a.page / a.block;
  const float* in = w.in ? w.in + (int64_t)h * a.nnz + s.pb : nullptr;
  float* out = w.out + (int64_t)h * a.nnz + s.pb;
  // where the units' statistics begin, their subtiles, and all of these
  int p0 = 0, units = a.n, span = spb, subs = a.n * spb;
  int64_t from = ((int64_t)b * a.hkv + h) * a.n * spb;
  if constexpr (!LISTED) {
    p0 = (int)((unsigned)(piece * a.ps + spp - 1) / (unsigned)spp);
    units = (piece == pc.n - 1 ? s.np : (int)((unsigned)((piece + 1) * a.ps + spp - 1) / (unsigned)spp)) - p0;
    span = spp;
    subs = subs_of(s) - p0 * spp;
    from = subs > 0 ? ((int64_t)h * a.nnz + s.pb + p0) * spp : 0;
  }
  const float2* stat = a.stat + from * group;
  const int top = max(subs - 1, 0);
  float2 y[NQ][4];
  auto fetch = [&](int u, int k0) {
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int sub = (u + 16 * q) * span + k0 + k;
        const bool there = u + 16 * q < units && k0 + k < span && sub < subs && l16 < group;
        // what is not there is read from the unit's own place (one address for all would hold up a channel of the L2)
        const float2 x = stat[(int64_t)min(sub, top) * group + min(l16, group - 1)];
        y[q][k] = make_float2(x.x, there ? x.y : 0.f);
      }
  };
  // s_page[j]: the page of listed block base + j - 1, -1 for none
  auto list_pages = [&](int base, int n) {
    const int* list = a.blocks + ((int64_t)b * a.hkv + h) * a.n;
    const int nblocks = blocks_of(s, a.block);
    for (int j = tid; j <= n; j += 256) {
      const int slot = base + j - 1, id = slot < 0 ? -1 : list[slot];
      const bool none_here = id < 0 || bad_block(id, slot ? list[slot - 1] : kNoPrev, nblocks);
      s_page[j] = none_here ? -1 : (int)((unsigned)id / (unsigned)bpp);
    }
  };
  // The listed blocks of one page follow each other: the first of them adds them all, so that a page is added to once.
  // (A list out of order may name a page again: hence the atomic.) A page whose blocks straddle two rounds of the LDS is
  // finished by the round it begins in, which looks past its end.
  for (int base = 0;; base += kListLds - bpp) {
    const int end = LISTED ? min(a.n, base + kListLds) : units;  // the last bpp of a round only to finish pages
    int u = base + r16, k0 = 0;
    fetch(u, 0);
    if (LISTED) {
      __syncthreads();  // the round before has been read
      list_pages(base, end - base);
    }
    if (base == 0) {
      if (LISTED)
        for (int p = tid; p < s.np; p += 256) out[p] = in ? w.decay * in[p] : 0.f;  // what every page keeps
      join_pieces(t, ml, pc.n, group, s_part);
      t = join(join(s_part[0][l16], s_part[1][l16]), join(s_part[2][l16], s_part[3][l16]));
      t.y = t.y == 0.f ? 0.f : 1.0f / t.y;
    }
    float sum[NQ] = {};
    while (u < end) {
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          sum[q] += y[q][k].y == 0.f ? 0.f : y[q][k].y * __builtin_amdgcn_exp2f(y[q][k].x - t.x) * t.y;
      k0 += 4;
      if (k0 >= span) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const float x = group_sum<16>(sum[q]);
          const int unit = u + 16 * q;
          if (l16 == 0 && unit < end) {
            if (LISTED) s_share[unit - base] = x;
            else out[p0 + unit] = (in ? w.decay * in[p0 + unit] : 0.f) + x;
          }
          sum[q] = 0.f;
        }
        u += 16 * NQ;
        k0 = 0;
      }
      if (u < end) fetch(u, k0);
    }
    if (!LISTED) return;
    __syncthreads();
    const int n = end - base;
    for (int j = tid; j < (end < a.n ? n - bpp : n); j += 256) {
      const int page = s_page[j + 1];
      if (page < 0 || s_page[j] == page) continue;
      float x = 0.f;
      for (int k = j; k < n && s_page[k + 1] == page; ++k) x += s_share[k];
      atomicAdd(out + page, x);
    }
    if (end == a.n) return;
  }
}

// The first batch * hkv * split workgroups: output rows. The others: page weights. A merge is three dependent trips to
// memory: 4 us for one sequence's 64 pieces, 5.8 for 512 pieces of 8 sequences with their weights.
template <int D, bool LISTED>
__global__ __launch_bounds__(256) void paged_blocks_merge_kernel(const BlkArgs a, const WeightArgs w) {
  __shared__ float2 s_part[4][16];
  __shared__ axk_f32x4 s_o[4][64];
  __shared__ float s_share[LISTED ? kListLds : 1];
  __shared__ int s_page[LISTED ? kListLds + 1 : 1];
  const int rows = a.batch * a.hkv, x = (int)blockIdx.x - rows * w.split;
  int b, h, piece = 0;
  Pieces pc;
  Seq s;
  if (x < 0 || LISTED) {
    const int row = x < 0 ? blockIdx.x / w.split : x;
    b = row / a.hkv;
    h = row - b * a.hkv;
    s = seq_of(a.indptr, a.last, b, a.page, a.nnz);
    pc = {(int64_t)row * a.pieces, a.pieces};
    if (!LISTED) {
      const int before = (int)min((unsigned)pieces_before(a, b), (unsigned)a.pieces);
      pc = {(int64_t)h * a.pieces + before, min(pieces_of(s, a.ps), a.pieces - before)};
    }
    if (x < 0) {
      merge_output<D>(a, b, h, blockIdx.x - row * w.split, pc, s_part, s_o);
      return;
    }
  } else {  // one workgroup per piece, for the pages that begin in it
    h = x / a.pieces;
    const PieceOf p = find_piece(a, x - h * a.pieces);
    if (p.b >= a.batch) return;
    b = p.b;
    piece = p.piece;
    s = p.s;
    pc = {x - piece, min(pieces_of(s, a.ps), (h + 1) * a.pieces - (x - piece))};
  }
  merge_weights<LISTED>(a, w, b, h, piece, s, pc, s_part, s_share, s_page);
}

// ---- eviction ----
// One workgroup per sequence: its `budget` pages of largest weight (summed over the KV heads in 64 bits, so that the
// order of the sum does not decide), the first `first` and last `keep_last` always among them, in their order into the
// new table; the others' ids into `freed`. Every workgroup finds its places from the whole indptr, and fills as much of
// the arrays' tails as it moved elsewhere. Bound by the selection's latency: 64 sequences of up to 2048 pages 11.6 us
// (26 us while a thread summed its pages' heads one after the other).
constexpr int kEvict = 1024;  // threads
constexpr int kEvictTile = 4 * kEvict;
__global__ __launch_bounds__(kEvict) void paged_evict_kernel(const float* __restrict__ w, const int* __restrict__ indptr,
                                                             const int* __restrict__ indices,
                                                             int* __restrict__ out_indptr, int* __restrict__ out_indices,
                                                             float* __restrict__ out_w, int* __restrict__ freed, int nnz,
                                                             int batch, int hkv, int budget, int first, int keep_last) {
  __shared__ PickLds<uint64_t, kEvict> lds;
  __shared__ unsigned s_sum[4][kEvict / 64];
  __shared__ int s_list[kEvictTile];  // a tile's pages: the kept ones from the front, the others from the back
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
  auto ptr = [&](int i) { return min(max(indptr[i], 0), nnz); };
  // kept and evicted pages of the sequences before b, and kept and all pages of all of them. (Unsigned, as every place made
  // of them is checked: where offsets of indptr fall back, the sums can be anything.)
  unsigned n4[4] = {0, 0, 0, 0};
  for (int i = tid; i < batch; i += kEvict) {
    const unsigned n = max(ptr(i + 1) - ptr(i), 0), k = min(n, (unsigned)budget);
    if (i < b) {
      n4[0] += k;
      n4[1] += n - k;
    }
    n4[2] += k;
    n4[3] += n;
  }
  const int waves = (min(batch, kEvict) + 63) / 64;  // that had sequences to add
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    n4[i] = (unsigned)wave_total((int)n4[i]);
    if (lane == 0) s_sum[i][wave] = n4[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    n4[i] = 0;
    for (int j = 0; j < waves; ++j) n4[i] += s_sum[i][j];
  }
  const unsigned kept = n4[0], gone = n4[1], all = n4[2], total = n4[3], table = (unsigned)nnz;
  const int pb = ptr(b), np = max(ptr(b + 1) - pb, 0), keep = min(np, budget);
  if (tid == 0) {
    if (b == 0) out_indptr[0] = 0;
    out_indptr[b + 1] = (int)(kept + keep);
  }
  // pages from[0 .. n) of the sequence (a null list: base, base + 1, ...) to places `at` onwards
  auto keep_pages = [&](const int* from, int base, int n, int at) {
    for (int i = tid; i < n; i += kEvict) {
      const int src = pb + (from ? from[i] : base + i);
      const unsigned dst = kept + at + i;
      if (dst >= table) break;
      out_indices[dst] = indices[src];
#pragma unroll 4
      for (int h = 0; h < hkv; ++h) out_w[(int64_t)h * nnz + dst] = w[(int64_t)h * nnz + src];
    }
  };
  if (np <= budget) {
    keep_pages(nullptr, 0, np, 0);
  } else {
    keep_pages(nullptr, 0, first, 0);
    keep_pages(nullptr, np - keep_last, keep_last, budget - keep_last);
    const int want = budget - first - keep_last, count = np - first - keep_last;
    if (want == 0) {
      for (int i = tid; i < count; i += kEvict)
        if (gone + i < table) freed[gone + i] = indices[pb + first + i];
    } else {
      int done0 = 0;  // pages kept in the tiles before
      auto keys = [&](int at, int n, auto& key) {
        constexpr int K = sizeof(key) / sizeof(uint64_t);
        double x[K];
#pragma unroll
        for (int i = 0; i < K; ++i) x[i] = 0.0;
        const float* row = w + pb + first + at;
        for (int h0 = 0; h0 < hkv; h0 += 4) {  // four heads' loads under way together
          float y[4][K];
#pragma unroll
          for (int h = 0; h < 4; ++h) load_run<K>(row + (int64_t)(h0 + h) * nnz, h0 + h < hkv ? n : 0, y[h]);
#pragma unroll
          for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < K; ++i) x[i] += (double)y[h][i];
        }
#pragma unroll
        for (int i = 0; i < K; ++i) key[i] = order_key(x[i]);
      };
      auto list = [&](int i, bool taken, int rank) {
        const int at = i & (kEvictTile - 1), k = rank - done0;
        s_list[taken ? k : kEvictTile - 1 - (at - k)] = first + i;
      };
      auto move = [&](int base, int n, int k) {
        __syncthreads();
        keep_pages(s_list, 0, k, first + done0);
        for (int i = tid; i < n - k; i += kEvict) {
          const unsigned dst = gone + base - done0 + i;
          if (dst < table) freed[dst] = indices[pb + s_list[kEvictTile - 1 - i]];
        }
        done0 += k;
        __syncthreads();
      };
      // a tile is at most as long as the list
      if (count <= kEvict) pick_largest<uint64_t, kEvict, 1>(count, want, keys, list, move, lds);
      else pick_largest<uint64_t, kEvict, 4>(count, want, keys, list, move, lds);
    }
  }
  // the tails: [all, nnz) of the table and of the weights, [total - all, nnz) of freed. A sequence's share of the first
  // is as long as what it evicted, of the second as what it kept; the last one also fills what no sequence had
  const int extra = b == batch - 1 && total < table ? (int)(table - total) : 0;
  for (int i = tid; i < np - keep + extra; i += kEvict) {
    const unsigned at = all + gone + i;
    if (at >= table) break;
    out_indices[at] = -1;
    for (int h = 0; h < hkv; ++h) out_w[(int64_t)h * nnz + at] = 0.f;
  }
  for (int i = tid; i < keep + extra; i += kEvict) {
    const unsigned at = total - all + kept + i;
    if (at < table) freed[at] = -1;
  }
}

}  // namespace

namespace {

constexpr int64_t kMaxSubs = 1 << 30;  // subtiles of a page table, or of a row's listed blocks: sums of them fit 32 bits

// Arrays that a call writes overlap neither what it reads nor each other.
struct Span {
  const void* p;
  size_t n;
};
template <int W, int R>
bool disjoint(const Span (&writes)[W], const Span (&reads)[R]) {
  for (int i = 0; i < W; ++i) {
    for (const Span& r : reads)
      if (axk_overlap(writes[i].p, writes[i].n, r.p, r.n)) return false;
    for (int j = 0; j < i; ++j)
      if (axk_overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n)) return false;
  }
  return true;
}

// Whether a dimension of a launch holds these workgroups: its threads are counted in 32 bits.
bool launch_fits(int64_t workgroups, int threads) { return workgroups <= (int64_t)0xffffffff / threads; }

int check_blocks(int64_t batch, int64_t hkv, int64_t d, int64_t page_size, int64_t block, int64_t num_pages, int64_t nnz) {
  AXK_REQUIRE(batch > 0 && batch <= (1 << 20) && hkv > 0 && hkv <= 4096, AXK_E_SHAPE);
  AXK_REQUIRE(d == 64 || d == 128 || d == 256, AXK_E_SHAPE);
  AXK_REQUIRE(page_size >= kSub && page_size % kSub == 0 && page_size <= 4096, AXK_E_SHAPE);
  AXK_REQUIRE(block >= kSub && block % kSub == 0 && page_size % block == 0, AXK_E_SHAPE);
  AXK_REQUIRE(num_pages > 0 && nnz >= 0 && nnz * (page_size / kSub) <= kMaxSubs, AXK_E_SHAPE);
  return AXK_OK;
}

// The stored type of a cache by its dtype code (kBf16 or kFp8, the latter with a power-of-two scale); negative: refused.
int cache_type(int kv_dtype, float kv_scale) {
  if (kv_dtype == AXK_DT_BF16) return kBf16;
  if (kv_dtype != AXK_DT_FP8E4M3) return -AXK_E_DTYPE;
  int e = 0;
  const float m = frexpf(kv_scale, &e);
  return kv_scale > 0.f && m == 0.5f && e >= -125 && e <= 126 ? kFp8 : -AXK_E_SHAPE;
}

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

// How a decode over blocks is cut, from what the host knows: pieces of at least 128 tokens, so that each wave has a step,
// and of at most 2048; otherwise as many as run at once at D = 256, two workgroups a CU, since a second round would pay the
// lookups again. (Smaller heads leave room for more workgroups; their cut has not been measured apart.)
constexpr int64_t kPieces = 512;
struct BlkPlan {
  int ps, pieces;
  int split;            // workgroups of the merge that share a row's output, four values a lane
  bool direct;
  bool fits;            // both launches
  size_t ml, po, stat;  // bytes of each workspace part
};
BlkPlan blk_plan(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t page, int64_t nnz, int64_t block, int64_t n,
                 bool weights) {
  const int64_t rows = batch * hkv, group = hq / hkv;
  const int64_t subs = n ? n * (block / kSub) : nnz * (page / kSub);  // of a row, or of a KV head
  const int64_t heads = n ? rows : hkv;
  int64_t cut = kPieces / heads;  // pieces of a row, or of a KV head, less the partial ones that sequences end in
  if (!n) cut = cut - batch >= cut / 2 ? cut - batch : cut / 2;
  int64_t ps = cut > 1 ? ((subs + cut - 1) / cut + 7) / 8 * 8 : kMaxPs;
  ps = ps < 8 ? 8 : ps > kMaxPs ? kMaxPs : ps;
  BlkPlan p;
  p.ps = (int)ps;
  p.pieces = (int)((subs + ps - 1) / ps + (n ? 0 : batch));  // a sequence's last piece may be a partial one
  p.direct = n && p.pieces == 1 && !weights;
  const size_t items = (size_t)(n ? rows : hkv) * p.pieces;
  p.ml = p.direct ? 0 : round256(items * group * sizeof(float2));
  p.po = p.direct ? 0 : round256(items * group * d * sizeof(float));
  p.stat = weights ? round256((size_t)(n ? rows : hkv) * subs * group * sizeof(float2)) : 0;
  p.split = (int)((group * d / 4 + 63) / 64);
  p.fits = launch_fits(n ? rows * p.pieces : p.pieces, 256) &&
           (p.direct || launch_fits(rows * p.split + (weights ? (n ? rows : hkv * p.pieces) : 0), 256));
  return p;
}

template <int D>
int launch_blocks(const BlkArgs& a, const WeightArgs& w, int type, hipStream_t st) {
  const dim3 grid = a.blocks ? dim3((unsigned)(a.batch * a.hkv * a.pieces)) : dim3((unsigned)a.pieces, (unsigned)a.hkv);
  if (type == kI8) hipLaunchKernelGGL((paged_blocks_kernel<D, kI8>), grid, dim3(256), (BlkCfg<D, kI8>::LDS), st, a);
  else if (type == kFp8) hipLaunchKernelGGL((paged_blocks_kernel<D, kFp8>), grid, dim3(256), (BlkCfg<D, kFp8>::LDS), st, a);
  else hipLaunchKernelGGL((paged_blocks_kernel<D, kBf16>), grid, dim3(256), (BlkCfg<D, kBf16>::LDS), st, a);
  if (!a.direct) {
    const int64_t wgs = (int64_t)a.batch * a.hkv * w.split + (w.out ? (a.blocks ? (int64_t)a.batch : a.pieces) * a.hkv : 0);
    if (a.blocks) hipLaunchKernelGGL((paged_blocks_merge_kernel<D, true>), dim3((unsigned)wgs), dim3(256), 0, st, a, w);
    else hipLaunchKernelGGL((paged_blocks_merge_kernel<D, false>), dim3((unsigned)wgs), dim3(256), 0, st, a, w);
  }
  return axk_launch_status();
}

}  // namespace

namespace {

int kv_write_bounds(const uint16_t* k, const uint16_t* v, void* kv_cache, int type, float kv_scale, uint16_t* kv_scales,
                    uint16_t* bounds, const int32_t* loc, int64_t rows, int64_t hkv, int64_t d, int64_t page_size,
                    int64_t block_size, int64_t num_pages, int32_t* status, axk_stream_t stream) {
  AXK_REQUIRE(k && v && kv_cache && bounds && loc && (kv_scales || type != kI8), AXK_E_NULL);
  const int rc = check_blocks(1, hkv, d, page_size, block_size, num_pages, 0);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(rows >= 0 && rows <= kMaxRows, AXK_E_SHAPE);
  if (type < 0) return -type;
  AXK_REQUIRE(axk_aligned(k, 16) && axk_aligned(v, 16) && axk_aligned(kv_cache, 16) && axk_aligned(bounds, 16) &&
                  axk_aligned(kv_scales, 2),
              AXK_E_ALIGN);
  const size_t row = (size_t)hkv * d, slots = (size_t)num_pages * page_size * 2;
  const Span writes[] = {{kv_cache, slots * row * (type ? 1 : 2)},
                         {bounds, (size_t)num_pages * (page_size / block_size) * row * 4}, {kv_scales, slots * hkv * 2}};
  const Span reads[] = {{k, rows * row * 2}, {v, rows * row * 2}, {loc, (size_t)rows * 8}};
  AXK_REQUIRE(disjoint(writes, reads), AXK_E_ALIAS);
  if (rows == 0) return AXK_OK;
  AXK_LAUNCH_GATE();
  auto* fn = type == kI8 ? &paged_kv_write_bounds_kernel<kI8>
                         : type == kFp8 ? &paged_kv_write_bounds_kernel<kFp8> : &paged_kv_write_bounds_kernel<kBf16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)rows), dim3(256), 0, axk_stream(stream), k, v,
                     static_cast<unsigned char*>(kv_cache), kv_scales, bounds, loc, (int)rows, (int)hkv, (int)d,
                     (int)page_size, (int)block_size, num_pages, type == kFp8 ? kv_scale : 1.0f, status);
  return axk_launch_status();
}

int key_bounds(const void* kv_cache, int type, float kv_scale, const uint16_t* kv_scales, uint16_t* bounds,
               const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len, const int32_t* start,
               int64_t nnz, int64_t batch, int64_t hkv, int64_t d, int64_t page_size, int64_t block_size,
               int64_t num_pages, int32_t* status, axk_stream_t stream) {
  AXK_REQUIRE(kv_cache && bounds && indptr && (indices || nnz == 0) && last_page_len && (kv_scales || type != kI8),
              AXK_E_NULL);
  const int rc = check_blocks(batch, hkv, d, page_size, block_size, num_pages, nnz);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(launch_fits(nnz * (page_size / block_size), 256), AXK_E_SHAPE);
  if (type < 0) return -type;
  AXK_REQUIRE(axk_aligned(kv_cache, 16) && axk_aligned(bounds, 16) && axk_aligned(kv_scales, 2), AXK_E_ALIGN);
  const size_t row = (size_t)hkv * d, slots = (size_t)num_pages * page_size * 2;
  const size_t tb = (size_t)batch * 4;
  const Span writes[] = {{bounds, (size_t)num_pages * (page_size / block_size) * row * 4}};
  const Span reads[] = {{kv_cache, slots * row * (type ? 1 : 2)}, {kv_scales, slots * hkv * 2}, {indptr, tb + 4},
                        {indices, (size_t)nnz * 4}, {last_page_len, tb}, {start, tb}};
  AXK_REQUIRE(disjoint(writes, reads), AXK_E_ALIAS);
  if (nnz == 0) return AXK_OK;
  AXK_LAUNCH_GATE();
  auto* fn = type == kI8 ? &paged_key_bounds_kernel<kI8>
                         : type == kFp8 ? &paged_key_bounds_kernel<kFp8> : &paged_key_bounds_kernel<kBf16>;
  hipLaunchKernelGGL(fn, dim3((unsigned)(nnz * (page_size / block_size))), dim3(256), 0, axk_stream(stream),
                     static_cast<const unsigned char*>(kv_cache), kv_scales, bounds, indptr, indices, last_page_len, start,
                     (int)nnz, (int)batch, (int)hkv, (int)d, (int)page_size, (int)block_size, num_pages,
                     type == kFp8 ? 1.0f / kv_scale : 1.0f, status);
  return axk_launch_status();
}

}  // namespace

extern "C" int axk_paged_kv_write_bounds(const uint16_t* k, const uint16_t* v, void* kv_cache, int kv_dtype,
                                         float kv_scale, uint16_t* bounds, const int32_t* cache_location, int64_t rows,
                                         int64_t num_kv_heads, int64_t head_dim, int64_t page_size, int64_t block_size,
                                         int64_t num_pages, int32_t* status, axk_stream_t stream) {
  return kv_write_bounds(k, v, kv_cache, cache_type(kv_dtype, kv_scale), kv_scale, nullptr, bounds, cache_location, rows,
                         num_kv_heads, head_dim, page_size, block_size, num_pages, status, stream);
}

extern "C" int axk_paged_kv_write_bounds_i8(const uint16_t* k, const uint16_t* v, int8_t* kv_cache, uint16_t* kv_scales,
                                            uint16_t* bounds, const int32_t* cache_location, int64_t rows,
                                            int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                            int64_t block_size, int64_t num_pages, int32_t* status,
                                            axk_stream_t stream) {
  return kv_write_bounds(k, v, kv_cache, kI8, 1.0f, kv_scales, bounds, cache_location, rows, num_kv_heads, head_dim,
                         page_size, block_size, num_pages, status, stream);
}

extern "C" int axk_paged_key_bounds(const void* kv_cache, int kv_dtype, float kv_scale, uint16_t* bounds,
                                    const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len,
                                    const int32_t* start, int64_t nnz, int64_t batch, int64_t num_kv_heads,
                                    int64_t head_dim, int64_t page_size, int64_t block_size, int64_t num_pages,
                                    int32_t* status, axk_stream_t stream) {
  return key_bounds(kv_cache, cache_type(kv_dtype, kv_scale), kv_scale, nullptr, bounds, indptr, indices, last_page_len,
                    start, nnz, batch, num_kv_heads, head_dim, page_size, block_size, num_pages, status, stream);
}

extern "C" int axk_paged_key_bounds_i8(const int8_t* kv_cache, const uint16_t* kv_scales, uint16_t* bounds,
                                       const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len,
                                       const int32_t* start, int64_t nnz, int64_t batch, int64_t num_kv_heads,
                                       int64_t head_dim, int64_t page_size, int64_t block_size, int64_t num_pages,
                                       int32_t* status, axk_stream_t stream) {
  return key_bounds(kv_cache, kI8, 1.0f, kv_scales, bounds, indptr, indices, last_page_len, start, nnz, batch,
                    num_kv_heads, head_dim, page_size, block_size, num_pages, status, stream);
}

extern "C" int axk_paged_block_scores(const uint16_t* q, const uint16_t* bounds, const int32_t* indptr,
                                      const int32_t* indices, const int32_t* last_page_len, float* scores, int64_t nnz,
                                      int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
                                      int64_t page_size, int64_t block_size, int64_t num_pages, int32_t* status,
                                      axk_stream_t stream) {
  AXK_REQUIRE(q && bounds && indptr && (nnz == 0 || (indices && scores)) && last_page_len, AXK_E_NULL);
  const int rc = check_blocks(batch, num_kv_heads, head_dim, page_size, block_size, num_pages, nnz);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(num_qo_heads > 0 && num_qo_heads % num_kv_heads == 0 && num_qo_heads / num_kv_heads <= kMaxGroup, AXK_E_SHAPE);
  const int64_t total = nnz * (page_size / block_size), units = (total + 15) / 16 * num_kv_heads;
  AXK_REQUIRE(launch_fits((units + 3) / 4, 256), AXK_E_SHAPE);
  AXK_REQUIRE(axk_aligned(q, 16) && axk_aligned(bounds, 16) && axk_aligned(scores, 4), AXK_E_ALIGN);
  if (nnz == 0) return AXK_OK;
  const size_t tb = (size_t)batch * 4;
  const Span writes[] = {{scores, (size_t)num_kv_heads * total * 4}};
  const Span reads[] = {{q, tb / 2 * num_qo_heads * head_dim},
                        {bounds, (size_t)num_pages * (page_size / block_size) * num_kv_heads * head_dim * 4},
                        {indptr, tb + 4}, {indices, (size_t)nnz * 4}, {last_page_len, tb}};
  AXK_REQUIRE(disjoint(writes, reads), AXK_E_ALIAS);
  AXK_LAUNCH_GATE();
  auto* fn = head_dim == 64 ? &paged_block_scores_kernel<64>
                            : head_dim == 128 ? &paged_block_scores_kernel<128> : &paged_block_scores_kernel<256>;
  hipLaunchKernelGGL(fn, dim3((unsigned)((units + 3) / 4)), dim3(256), 0, axk_stream(stream), q, bounds, indptr, indices,
                     last_page_len, scores, (int)nnz, (int)batch, (int)num_qo_heads, (int)num_kv_heads, (int)page_size,
                     (int)block_size, num_pages, (unsigned)units, status);
  return axk_launch_status();
}

extern "C" int axk_paged_select_blocks(const float* scores, const int32_t* indptr, const int32_t* last_page_len,
                                       int32_t* blocks, int64_t nnz, int64_t batch, int64_t num_kv_heads,
                                       int64_t page_size, int64_t block_size, int64_t num_select, int64_t first,
                                       int64_t keep_last, axk_stream_t stream) {
  AXK_REQUIRE((scores || nnz == 0) && indptr && last_page_len && blocks, AXK_E_NULL);
  const int rc = check_blocks(batch, num_kv_heads, 64, page_size, block_size, 1, nnz);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(num_select > 0 && num_select <= (1 << 24) && first >= 0 && keep_last >= 0 &&
                  first + keep_last <= num_select,
              AXK_E_SHAPE);
  const int64_t total = nnz * (page_size / block_size);
  const bool small = total <= 2048;  // every row at most eight keys a thread of 256
  AXK_REQUIRE(launch_fits(batch * num_kv_heads, small ? 256 : 1024), AXK_E_SHAPE);
  AXK_REQUIRE(axk_aligned(scores, 4) && axk_aligned(blocks, 4), AXK_E_ALIGN);
  const size_t tb = (size_t)batch * 4;
  const Span writes[] = {{blocks, tb * num_kv_heads * num_select}};
  const Span reads[] = {{scores, (size_t)num_kv_heads * total * 4}, {indptr, tb + 4}, {last_page_len, tb}};
  AXK_REQUIRE(disjoint(writes, reads), AXK_E_ALIAS);
  AXK_LAUNCH_GATE();
  const dim3 grid((unsigned)(batch * num_kv_heads));
  if (small)
    hipLaunchKernelGGL(paged_select_blocks_kernel<256>, grid, dim3(256), 0, axk_stream(stream), scores, indptr,
                       last_page_len, blocks, (int)nnz, (int)num_kv_heads, (int)page_size, (int)block_size,
                       (int)num_select, (int)first, (int)keep_last);
  else
    hipLaunchKernelGGL(paged_select_blocks_kernel<1024>, grid, dim3(1024), 0, axk_stream(stream), scores, indptr,
                       last_page_len, blocks, (int)nnz, (int)num_kv_heads, (int)page_size, (int)block_size,
                       (int)num_select, (int)first, (int)keep_last);
  return axk_launch_status();
}

extern "C" size_t axk_paged_decode_blocks_workspace_size(int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads,
                                                         int64_t head_dim, int64_t page_size, int64_t nnz,
                                                         int64_t block_size, int64_t num_select, int with_weights) {
  if (check_blocks(batch, num_kv_heads, head_dim, page_size, num_select ? block_size : kSub, 1, nnz) != AXK_OK) return 0;
  if (num_qo_heads <= 0 || num_qo_heads % num_kv_heads || num_qo_heads / num_kv_heads > kMaxGroup) return 0;
  if (num_select < 0 || num_select > kMaxSubs || num_select * (block_size / kSub) > kMaxSubs) return 0;
  const BlkPlan p = blk_plan(batch, num_qo_heads, num_kv_heads, head_dim, page_size, nnz, block_size, num_select,
                             with_weights != 0);
  return p.fits ? p.ml + p.po + p.stat : 0;
}

namespace {

int decode_blocks(const uint16_t* q, const void* kv_cache, int type, float kv_scale, const uint16_t* kv_scales,
                  const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len, const int32_t* blocks,
                  int64_t block_size, int64_t num_select, uint16_t* out, const float* weights_in, float* weights_out,
                  float decay, int64_t nnz, int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
                  int64_t page_size, int64_t num_pages, float sm_scale, int32_t* status, void* workspace,
                  size_t workspace_bytes, axk_stream_t stream) {
  AXK_REQUIRE(q && kv_cache && indptr && (indices || nnz == 0) && last_page_len && out && (kv_scales || type != kI8),
              AXK_E_NULL);
  if (!blocks) {
    AXK_REQUIRE(num_select == 0, AXK_E_NULL);
    block_size = kSub;
  } else {
    AXK_REQUIRE(num_select > 0, AXK_E_SHAPE);
  }
  const int rc = check_blocks(batch, num_kv_heads, head_dim, page_size, block_size, num_pages, nnz);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(num_qo_heads > 0 && num_qo_heads % num_kv_heads == 0 && num_qo_heads / num_kv_heads <= kMaxGroup, AXK_E_SHAPE);
  AXK_REQUIRE(num_select <= kMaxSubs && num_select * (block_size / kSub) <= kMaxSubs, AXK_E_SHAPE);
  AXK_REQUIRE(!weights_in || weights_out, AXK_E_NULL);
  if (type < 0) return -type;
  AXK_REQUIRE(axk_aligned(q, 16) && axk_aligned(kv_cache, 16) && axk_aligned(out, 8) && axk_aligned(weights_in, 4) &&
                  axk_aligned(weights_out, 4) && axk_aligned(blocks, 4) && axk_aligned(kv_scales, 2),
              AXK_E_ALIGN);
  const bool weights = weights_out && nnz > 0;
  const BlkPlan p = blk_plan(batch, num_qo_heads, num_kv_heads, head_dim, page_size, nnz, block_size, num_select, weights);
  AXK_REQUIRE(p.fits, AXK_E_SHAPE);
  const size_t need = p.ml + p.po + p.stat;
  AXK_REQUIRE(!need || (workspace && workspace_bytes >= need && axk_aligned(workspace, 256)), AXK_E_WORKSPACE);
  // (The merge reads the page table and the lists again, after the first kernel has written the workspace.)
  const size_t tb = (size_t)batch * 4, qb = tb / 2 * num_qo_heads * head_dim, wb = (size_t)num_kv_heads * nnz * 4;
  const size_t slots = (size_t)num_pages * page_size * 2 * num_kv_heads;
  const Span writes[] = {{out, qb}, {weights_out, wb}, {workspace, need}};
  const Span reads[] = {{q, qb}, {kv_cache, slots * head_dim * (type ? 1 : 2)}, {kv_scales, slots * 2}, {indptr, tb + 4},
                        {indices, (size_t)nnz * 4}, {last_page_len, tb}, {blocks, tb * num_kv_heads * num_select},
                        {weights_in == weights_out ? nullptr : weights_in, wb}};
  AXK_REQUIRE(disjoint(writes, reads), AXK_E_ALIAS);
  BlkArgs a;
  a.q = q;
  a.cache = static_cast<const unsigned char*>(kv_cache);
  a.indptr = indptr;
  a.indices = indices;
  a.last = last_page_len;
  a.blocks = blocks;
  a.n = (int)num_select;
  a.block = (int)block_size;
  a.nnz = (int)nnz;
  a.batch = (int)batch;
  a.hq = (int)num_qo_heads;
  a.hkv = (int)num_kv_heads;
  a.page = (int)page_size;
  a.num_pages = num_pages;
  a.kv_scales = kv_scales;
  a.scale = sm_scale * kLog2e;
  a.inv_scale = type == kFp8 ? 1.0f / kv_scale : 1.0f;
  a.ps = p.ps;
  a.pieces = p.pieces;
  a.direct = p.direct;
  a.out = out;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  a.ml = p.direct ? nullptr : reinterpret_cast<float2*>(ws);
  a.po = p.direct ? nullptr : reinterpret_cast<float*>(ws + p.ml);
  a.stat = weights ? reinterpret_cast<float2*>(ws + p.ml + p.po) : nullptr;
  a.status = status;
  if (head_dim == 256 && type == kBf16) {  // 64 KiB of dynamic LDS beside the static: to be allowed once on each device
    static AxkOnce once[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return AXK_E_LAUNCH;
    if (const int e = axk_raise_lds(once[dev & 63], reinterpret_cast<const void*>(&paged_blocks_kernel<256, kBf16>),
                                    BlkCfg<256, kBf16>::LDS))
      return e;
  }
  const WeightArgs w = {weights_in, weights ? weights_out : nullptr, decay, p.split};
  AXK_LAUNCH_GATE();
  switch (head_dim) {
    case 64: return launch_blocks<64>(a, w, type, axk_stream(stream));
    case 128: return launch_blocks<128>(a, w, type, axk_stream(stream));
    default: return launch_blocks<256>(a, w, type, axk_stream(stream));
  }
}

}  // namespace

extern "C" int axk_paged_decode_blocks(const uint16_t* q, const void* kv_cache, int kv_dtype, float kv_scale,
                                       const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len,
                                       const int32_t* blocks, int64_t block_size, int64_t num_select, uint16_t* out,
                                       const float* weights_in, float* weights_out, float decay, int64_t nnz,
                                       int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
                                       int64_t page_size, int64_t num_pages, float sm_scale, int32_t* status,
                                       void* workspace, size_t workspace_bytes, axk_stream_t stream) {
  return decode_blocks(q, kv_cache, cache_type(kv_dtype, kv_scale), kv_scale, nullptr, indptr, indices, last_page_len,
                       blocks, block_size, num_select, out, weights_in, weights_out, decay, nnz, batch, num_qo_heads,
                       num_kv_heads, head_dim, page_size, num_pages, sm_scale, status, workspace, workspace_bytes, stream);
}

extern "C" int axk_paged_decode_blocks_i8(const uint16_t* q, const int8_t* kv_cache, const uint16_t* kv_scales,
                                          const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len,
                                          const int32_t* blocks, int64_t block_size, int64_t num_select, uint16_t* out,
                                          const float* weights_in, float* weights_out, float decay, int64_t nnz,
                                          int64_t batch, int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim,
                                          int64_t page_size, int64_t num_pages, float sm_scale, int32_t* status,
                                          void* workspace, size_t workspace_bytes, axk_stream_t stream) {
  return decode_blocks(q, kv_cache, kI8, 1.0f, kv_scales, indptr, indices, last_page_len, blocks, block_size, num_select,
                       out, weights_in, weights_out, decay, nnz, batch, num_qo_heads, num_kv_heads, head_dim, page_size,
                       num_pages, sm_scale, status, workspace, workspace_bytes, stream);
}

extern "C" int axk_paged_evict_pages(const float* weights, const int32_t* indptr, const int32_t* indices,
                                     int32_t* out_indptr, int32_t* out_indices, float* out_weights, int32_t* freed,
                                     int64_t nnz, int64_t batch, int64_t num_kv_heads, int64_t budget, int64_t first,
                                     int64_t keep_last, axk_stream_t stream) {
  AXK_REQUIRE(indptr && out_indptr && (nnz == 0 || (weights && indices && out_indices && out_weights && freed)), AXK_E_NULL);
  AXK_REQUIRE(batch > 0 && batch <= (1 << 20) && num_kv_heads > 0 && num_kv_heads <= 4096 && nnz >= 0 && nnz <= 0x3fffffff,
              AXK_E_SHAPE);
  AXK_REQUIRE(first >= 0 && keep_last >= 1 && budget >= first + keep_last && budget <= 0x3fffffff, AXK_E_SHAPE);
  const size_t ib = (size_t)nnz * 4, pb = (size_t)(batch + 1) * 4, wb = (size_t)num_kv_heads * nnz * 4;
  AXK_REQUIRE(axk_aligned(out_indptr, 4) && axk_aligned(out_indices, 4) && axk_aligned(out_weights, 4) && axk_aligned(freed, 4),
              AXK_E_ALIGN);
  const Span writes[] = {{out_indptr, pb}, {out_indices, ib}, {out_weights, wb}, {freed, ib}};
  const Span reads[] = {{weights, wb}, {indptr, pb}, {indices, ib}};
  AXK_REQUIRE(disjoint(writes, reads), AXK_E_ALIAS);
  AXK_LAUNCH_GATE();
  hipLaunchKernelGGL(paged_evict_kernel, dim3((unsigned)batch), dim3(kEvict), 0, axk_stream(stream), weights, indptr, indices,
                     out_indptr, out_indices, out_weights, freed, (int)nnz, (int)batch, (int)num_kv_heads, (int)budget,
                     (int)first, (int)keep_last);
  return axk_launch_status();
}
