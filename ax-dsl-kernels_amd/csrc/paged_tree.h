// Attention of a tree of drafted tokens over a paged KV cache (paged_tree_*.hip instantiate it per stored type).
//
// The cache and page table are those of paged_attn.hip. A sequence's tree is parents[b, t], t < T <= 64: the node's parent (a
// node before it), -1 (the last token of the history) or -2 (no node). The n nodes' K / V are the last n cached tokens, node t
// at position len - n + t. For query head g of KV head h, with A(t) node t and its ancestors,
//   o_tg = sum_j p_j v_j,  p = softmax over {history} + A(t) of scale q_tg . k_j.
//
// The rows of one (sequence, KV head) are r = t G + g (G query heads a KV head): a workgroup takes 32 RT WR of them and a piece
// of the sequence's tokens, in pairs of 16-token tiles (a tile never leaves its page). Its four waves are WR row slices times
// KG = 4 / WR token groups; a group keeps K and V of its pairs in LDS as they are stored, in rings filled by direct loads, and
// every wave computes S^T = K Q^T (32 tokens x its 32 RT rows) and O^T += V^T P^T over the whole head dim on 32x32x16 MFMA. In
// S^T's layout a lane holds 16 of its row's scores, which as bf16 are P^T's operand as they stand: no exchange, and the softmax's
// maximum and sum cost one exchange with lane + 32. K is scored one pair ahead of V, so that the exponentials of one pair run
// beside the products of the next.
//
// Roundings: P to bf16 for the product with V (2^-8 of each weight, the only one beside the output's own), E4M3 and int8 values
// are exact in bf16; scores, maxima, sums, O and the pieces' partials are fp32. The maximum that weights refer to follows the
// scores only in steps of more than 2^8, which rescales O rarely and changes no bit of what is represented.
//
// What bounds it. Few rows: the start and the end of a piece (lookup, first page, first pair, join), run once and waiting for 57%
// of the time: one draft of 8 nodes, pieces of four pairs, takes 16.6 us and a merge of 7. Many rows: a wave's instructions, not
// the matrix cores: one wave a SIMD (O and Q take 3 RT D / 4 of its registers) issues 381 instructions a pair in the loop without
// masks, of which 32 are MFMAs; it issues in 58% of its cycles and waits in 30, its matrix core works in 42. 8 sequences of 32768
// tokens x 64 nodes x 32 heads of 256: 565-580 us a replay, 620-630 TFLOP/s, HBM read 1.1 times (a KV head's row blocks read a
// piece through one L2). Its nodes fill 25 of 32 blocks; cutting the work into equal shares of the 25 measured the same time (594
// and 611 us), with twice the partials.
#pragma once
#include "axk_common.h"
#include "axk_host.h"
#include "axk_tree_common.h"

namespace axk_tree {

typedef int axk_i32x4 __attribute__((ext_vector_type(4)));

enum { kBf16 = AXK_KV_BF16, kFp8 = AXK_KV_FP8, kI8 = AXK_KV_I8 };
constexpr int kTile = 16;
constexpr int kPair = 32;
constexpr int kMergeRows = 4;           // rows (waves) of a merge workgroup
constexpr float kLog2e = 1.4426950408889634f;

struct TreeArgs {
  const uint16_t* q;            // [B, T, HQ, D]
  const unsigned char* cache;   // [P, 2, page, HKV, D]
  const uint16_t* scales;       // int8: [P, 2, page, HKV]
  const int *indptr, *indices, *last, *parents;
  uint16_t* out;                // [B, T, HQ, D]
  float2* ml;                   // a piece's (maximum, sum) of each row, and its unnormalised output
  float* po;
  int* status;
  int batch, nodes, hq, hkv, page, nnz;
  int nb;                       // row blocks of a (sequence, KV head)
  int den, min_piece;           // pieces that all sequences share, and a piece's least pairs
  int groups;                   // upper bound of pieces x KV heads
  int split;                    // whether a sequence may have several pieces
  int64_t num_pages;
  float scale, inv_scale;       // softmax scale * log2(e); 1 / kv_scale
};

// Sequence b of the page table. Offsets outside the table and a last page longer than a page are clamped, so that no index
// built from them leaves its array.
struct Seq {
  int pb, np, len;
};
AXK_DEV Seq seq_from(int lo, int hi, int last, int page, int nnz) {
  Seq s;
  s.pb = min(max(lo, 0), nnz);
  s.np = min(max(hi, s.pb), nnz) - s.pb;
  s.len = s.np ? (s.np - 1) * page + min(max(last, 0), page) : 0;  // nnz * page < 2^31
  return s;
}
AXK_DEV int pairs_of(const Seq& s) { return (s.len + kPair - 1) / kPair; }

// A batch of more sequences is not cut: it fills the device by its number, and looking a piece up among its sequences would cost
// more than the rounds that long ones stand out by. Us with and without, 2 heads of 128: 512 sequences of up to 1000 tokens 121
// and 67, 1000 of them 313 and 137; 48 sequences of up to 2000 tokens (2 heads of 256) 38 and 49.
constexpr int kSplitBatch = 256;

// How the batch is cut: every sequence into pieces of P pairs, P such that the pieces of all row blocks and KV heads run at
// once: total / den pairs, or up to twice as many, if no more than den pieces come out so (65 sequences of 1000 to 8000 tokens,
// 2 heads of 256: 128 us, with total / den 167). Else P is total / den, and pieces follow one another: short sequences are pieces
// of their own, and a P that keeps their number down leaves a long one whole (131072 tokens beside 63 of 200, 8 heads of 256:
// 248 us, as one piece 3480). There are at most den + batch. Where the first P would cut the longest sequence once and not far
// from its end, all are left whole: 128 sequences of 500 to 1000 tokens, 4 nodes x 16 heads of 256, 55 us with the cut and 52
// without. Every wave of both launches derives the same cut from the page table: the total is a float sum in a fixed order.
struct Piece {
  int b;       // sequence (-1: none)
  int j, ns;   // piece of the sequence, and how many it has
  int first;   // the sequence's first piece among all
  int size;    // P
  Seq s;
};
// By piece (`by_piece`: `want` counts all pieces) or by sequence (`want` is b).
AXK_DEV Piece find_piece(const TreeArgs& a, int want, bool by_piece, int kg) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = 0, tail = 0;
  auto load = [&](int b0) {
    const int at = min(b0 + lane, a.batch - 1);
    lo = a.indptr[at];
    hi = a.indptr[at + 1];
    tail = a.last[at];
  };
  if (!a.split) {  // a piece a sequence: nothing to look for
    const int b = min(want, a.batch - 1);
    Piece k;
    k.b = want < a.batch ? b : -1;
    k.j = 0, k.ns = 1, k.first = b, k.size = 0x40000000;
    k.s = seq_from(a.indptr[b], a.indptr[b + 1], a.last[b], a.page, a.nnz);
    return k;
  }
  float total = 0.f, longest = 0.f;
  float pairs[kSplitBatch / 64];  // of sequences lane, lane + 64, .., less one half
#pragma unroll
  for (int i = 0; i < kSplitBatch / 64; ++i) {
    pairs[i] = -0.5f;
    if (i && a.batch <= 64 * i) continue;
    load(64 * i);
    const float n = 64 * i + lane < a.batch ? (float)pairs_of(seq_from(lo, hi, tail, a.page, a.nnz)) : 0.f;
    pairs[i] += n;
    total += wave_sum(n);
    longest = fmaxf(longest, wave_max(n));
  }
  int p = max(a.min_piece, (int)fminf(total / (float)a.den, 0x1p28f) + 1);  // (offsets that fall back may add up to any total)
  if (longest <= 1.5f * (float)p) p = max(p, (int)longest);  // sequences even enough to be left whole
  auto whole_groups = [&](int x) { return (x + kg - 1) / kg * kg; };
  // How many pieces: n / size rounded up is (n - 1/2) / size rounded down, and 1 (to 2^21 pairs a sequence; beyond, the number
  // may be off by one, which changes the cut, not its bound).
  auto pieces = [&](int size) {
    const float each = __builtin_amdgcn_rcpf((float)size);
    int n = 0;
#pragma unroll
    for (int i = 0; i < kSplitBatch / 64; ++i)
      if (!i || a.batch > 64 * i) n += 64 * i + lane < a.batch ? (int)(pairs[i] * each) + 1 : 0;
    return __builtin_amdgcn_readlane(wave_scan(n), 63);
  };
  Piece k;
  k.b = -1;
  k.size = whole_groups(p);
  const int most = 2 * k.size;
  int n = a.batch <= a.den ? pieces(k.size) : 0;  // (a sequence is at least a piece)
  // (up to den / 2 sequences no size has to be tried: with the most, full pieces and last ones are den / 2 each)
  if (n > a.den && (2 * a.batch <= a.den || pieces(most) <= a.den))
    for (int i = 0; i < 8 && n > a.den; ++i) {
      const int more = whole_groups((int)((float)k.size * (float)n / (float)a.den) + 1);
      k.size = i < 7 ? min(more, most) : most;
      if (k.size == most) break;
      n = pieces(k.size);
    }
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) load(b0);
    // (at least one each, which writes the zeros of a sequence without tokens)
    const int here = pairs_of(seq_from(lo, hi, tail, a.page, a.nnz));
    const int mine = b0 + lane < a.batch ? max(1, (int)((unsigned)(here + k.size - 1) / (unsigned)k.size)) : 0;
    const int incl = wave_scan(mine), excl = base + incl - mine;
    const bool found = by_piece ? want >= excl && want < excl + mine : b0 + lane == want;
    const uint64_t hit = __ballot(found);
    if (hit) {
      const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)hit) - 1);
      k.b = b0 + src;
      k.ns = __builtin_amdgcn_readlane(mine, src);
      k.first = __builtin_amdgcn_readlane(excl, src);
      k.j = by_piece ? want - k.first : 0;
      k.s = seq_from(__builtin_amdgcn_readlane(lo, src), __builtin_amdgcn_readlane(hi, src),
                     __builtin_amdgcn_readlane(tail, src), a.page, a.nnz);
      return k;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return k;
}

// RT row tiles of 32 a wave, WR waves over the rows and KG = 4 / WR over the tokens.
template <int D, int T, int RT, int WR>
struct TreeCfg {
  static constexpr int KG = 4 / WR;
  static constexpr int RB = 32 * RT * WR;          // rows of a workgroup
  static constexpr int KS = D / 16;                // 16-deep MFMA steps of Q K^T
  static constexpr int DT = D / 32;                // 32-wide tiles of O
  static constexpr int RBY = T == kBf16 ? 2 * D : D;  // bytes of a stored row
  static constexpr int NCH = RBY / 16;             // its 16-byte chunks
  static constexpr int RPI = 1024 / RBY;           // rows of one direct-to-LDS instruction (64 lanes x 16 B)
  static constexpr int IPP = kTile / RPI;          // instructions of a tile's K (or V)
  static constexpr int IPW = 4 * IPP / WR;         // a wave's, of a pair
  static constexpr int TILE = kTile * RBY, PLANE = 2 * TILE;
  static constexpr int OCC = RT == 1 && D <= 128 ? 2 : 1;  // workgroups a CU (registers: Q and O take 3 RT D / 4 of a wave's)
  // Pairs of K, and of V, that a group holds in LDS: K is scored one pair ahead of the V that is weighted.
  static constexpr int LDS_MAX = (OCC == 2 ? 80 : 160) * 1024 - 4096;
  static constexpr int NS = KG * 8 * PLANE <= LDS_MAX ? 4 : 2;
  static constexpr int SCALES = T == kI8 ? 8 * 256 : 0;  // a group's scales: of eight pairs' K and V rows
  static constexpr int GROUP = 2 * NS * PLANE + SCALES;
  static constexpr int RING = KG * GROUP;
  static constexpr int JOIN = KG == 2 ? WR * RT * 32 * (D * 4 + 8) : 0;  // one group's results
  static constexpr int LDS = (RING > JOIN ? RING : JOIN) + kMaxNodes * 8 + 16;  // and the ancestors, and a flag
  static_assert(PLANE % (WR * 1024) == 0, "V is looked through by all of a group's waves");
  static_assert(KG * 4 * PLANE <= LDS_MAX && LDS <= 160 * 1024 && KG <= 2 && (NS == 2 || NS == 4), "LDS");
  // Where chunk c of a tile's row r is kept: K fragment reads (32 rows, one or two chunks each) and transposing V reads (4 rows
  // x 64 bytes of bf16, 8 rows x 32 bytes of 8 bits) then cover all LDS banks.
  static constexpr __host__ __device__ int kswz(int r) { return NCH == 4 ? (r >> 1) & 3 : r & (NCH < 16 ? NCH - 1 : 15); }
  static constexpr __host__ __device__ int vswz(int r) {
    if constexpr (T == kBf16) return 4 * (NCH < 16 ? (r >> 1) & 1 : r & 3);
    return 2 * (NCH < 8 ? (r >> 1) & 1 : r & 3);
  }
};

// Eight stored 8-bit values (two dwords) as bf16: E4M3 times a power of two, or int8 codes, both exact.
template <int T>
AXK_DEV axk_bf16x8 bf16_of(uint32_t w0, uint32_t w1, float inv_scale) {
  axk_u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = i < 2 ? w0 : w1;
    if constexpr (T == kFp8)
      r[i] = __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, inv_scale, true)
                                                : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, inv_scale, false));
    else
      r[i] = pack_bf16x2((float)(int8_t)(x >> (16 * (i & 1))), (float)(int8_t)(x >> (16 * (i & 1) + 8)));
  }
  return __builtin_bit_cast(axk_bf16x8, r);
}

// A 2-byte value a lane, zero-extended, into LDS at lds_base + 4 * lane.
AXK_DEV void lds_dma2(const void* gptr, uint32_t lds_base_any) {
  const uint32_t lds_base = __builtin_amdgcn_readfirstlane(lds_base_any);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_ushort %1, off"
      :
      : "s"(lds_base), "v"(gptr)
      : "memory");
}

template <int D, int T, int RT, int WR>
__global__ __launch_bounds__(256, (TreeCfg<D, T, RT, WR>::OCC)) void paged_tree_kernel(TreeArgs a) {
  using C = TreeCfg<D, T, RT, WR>;
  constexpr int KG = C::KG, RB = C::RB, KS = C::KS, DT = C::DT, NS = C::NS;
  extern __shared__ __align__(16) unsigned char smem[];
  uint64_t* const s_anc = reinterpret_cast<uint64_t*>(smem + C::LDS - kMaxNodes * 8 - 16);
  volatile int* const s_odd = reinterpret_cast<int*>(smem + C::LDS - 16);  // whether V of a node held what is no number

  const int sl = blockIdx.x >> 3;
  const int gi = sl / a.nb * 8 + (blockIdx.x & 7), blk = sl % a.nb;
  if (gi >= a.groups) return;
  const int kvh = gi % a.hkv;
  const Piece k = find_piece(a, gi / a.hkv, true, KG);
  if (k.b < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / WR, wr = wave % WR;
  const int l16 = lane & 15, l32 = lane & 31, h = lane >> 5;
  const int group = a.hq / a.hkv, rows = a.nodes * group;

  const int parent = lane < a.nodes ? a.parents[(int64_t)k.b * a.nodes + lane] : -2;
  const int n = node_count(parent);
  const int base = k.s.len - n;  // the first node's position
  if (base < 0 && a.status && threadIdx.x == 0) *a.status = 1;
  if (blk * RB >= n * group) {  // no node of this block is one
    if (k.ns == 1)
      for (int i = threadIdx.x; i < RB * D / 8; i += 256) {
        const int rr = blk * RB + i / (D / 8);
        if (rr < rows) {
          const int t = rr / group;
          const int64_t at = (((int64_t)k.b * a.nodes + t) * a.hq + kvh * group + rr - t * group) * D + i % (D / 8) * 8;
          *reinterpret_cast<axk_u32x4*>(a.out + at) = axk_u32x4{0u, 0u, 0u, 0u};
        }
      }
    return;
  }

  // this lane's rows (lanes l and l + 32 share them), and their q as the B operand
  const float c = a.scale == 0.f ? 1.0f : fabsf(a.scale);
  // a negative scale moves into Q's signs and a zero scale into zero rows, so that scores keep their order
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, keep = a.scale != 0.f ? 0xffffffffu : 0u;
  int node[RT];
  int64_t qrow[RT];
  axk_bf16x8 qb[RT][KS];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = blk * RB + 32 * (RT * wr + t) + l32, rr = min(r, rows - 1);
    node[t] = r < rows ? r / group : -1;
    const int nd = rr / group;
    qrow[t] = ((int64_t)k.b * a.nodes + nd) * a.hq + kvh * group + rr - nd * group;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // element (h, j) of step s: channel 16 s + 8 h + j; 8-bit rows are read 16 bytes a lane, two steps at a time:
      // 32 (s / 2) + 16 h + 8 (s % 2) + j
      const int ch = T == kBf16 ? 16 * s + 8 * h : 32 * (s / 2) + 16 * h + 8 * (s % 2);
      axk_u32x4 w = *reinterpret_cast<const axk_u32x4*>(a.q + qrow[t] * D + ch);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = (w[e] ^ flip) & keep;
      qb[t][s] = __builtin_bit_cast(axk_bf16x8, w);
    }
  }

  // this group's pairs p_beg + kg, + KG, .. before p_end
  const int p_beg = k.j * k.size + kg, p_end = min(pairs_of(k.s), k.j * k.size + k.size);
  const int steps = p_end > p_beg ? (p_end - p_beg + KG - 1) / KG : 0;
  const int all_steps = (max(p_end - k.j * k.size, 0) + KG - 1) / KG;  // of the workgroup (kg = 0)
  const int tpp = a.page / kTile;
  const int64_t row_bytes = (int64_t)a.hkv * C::RBY, plane_bytes = (int64_t)a.page * row_bytes, tile_bytes = kTile * row_bytes;
  const unsigned char* const head0 = a.cache + (int64_t)kvh * C::RBY;

  // 64 pages of the sequence at a time: lane l holds the address of page 64 chunk + l; bad: the lanes whose page lies outside
  // the pool (they hold page 0's)
  int chunk = -1;
  uint32_t pg_lo = 0, pg_hi = 0, pg_id = 0;
  uint64_t bad = 0;
  auto set_chunk = [&](int ck) {
    chunk = ck;
    const int j = (ck << 6) + lane;
    int pid = j < k.s.np ? a.indices[k.s.pb + j] : 0;
    asm volatile("" : "+v"(pid));  // the compiler's wait for the load stays here, behind no loop of direct loads
    const bool out = pid < 0 || pid >= a.num_pages;
    bad = __ballot(out);
    if (bad && a.status && lane == 0) *a.status = 1;
    pg_id = out ? 0 : pid;
    const uint64_t at = (uint64_t)(uintptr_t)(head0 + (int64_t)pg_id * 2 * plane_bytes);
    pg_lo = (uint32_t)at;
    pg_hi = (uint32_t)(at >> 32);
  };
  // The cursor of K: the next pair's first tile and its page. This wave loads one tile of every pair (WR = 4: one plane of it).
  const int my_tile = WR == 4 ? wr >> 1 : wr, my_plane = wr & 1;
  int cur_lp = 2 * p_beg / tpp, cur_tp = 2 * p_beg - cur_lp * tpp, cur_p = p_beg;
  uint32_t bads = 0;  // two bits a pair in flight, the latest lowest: its tiles lie on pages outside the pool
  // That tile of the pair whose K is loaded next (k_), and of the one before it, whose V is (v_): its K (V lies plane_bytes
  // behind), its rows with tokens (none past the sequence or on a page outside the pool), and (int8) its first row in the
  // scales.
  const unsigned char *k_at = head0, *v_at = head0;
  int k_rows = 0, v_rows = 0;
  int64_t k_slot = 0;
  auto page_base = [&](int at) {
    const uint32_t lo = __builtin_amdgcn_readlane(pg_lo, at), hi = __builtin_amdgcn_readlane(pg_hi, at);
    return reinterpret_cast<const unsigned char*>((uintptr_t)(((uint64_t)hi << 32) | lo));
  };
  // Whether the next pair is whole and its pages are among those at hand.
  auto at_hand = [&]() {
    return (cur_lp >> 6) == chunk && ((cur_lp + (cur_tp + 1 == tpp)) >> 6) == chunk && cur_p * kPair + kPair <= k.s.len;
  };
  auto next_pair = [&](auto hot) {  // hot: at_hand() holds
    v_at = k_at, v_rows = k_rows;
    bads <<= 2;
    const int wrap = cur_tp + 1 == tpp, lp1 = cur_lp + wrap, tp1 = wrap ? 0 : cur_tp + 1;
    const int tok = cur_p * kPair + kTile * my_tile;
    int lp = my_tile ? lp1 : cur_lp, tp = my_tile ? tp1 : cur_tp;
    k_rows = decltype(hot)::value ? kTile : min(kTile, k.s.len - tok);
    uint32_t bad2;
    if (decltype(hot)::value || ((cur_lp >> 6) == chunk && (lp1 >> 6) == chunk)) {
      bad2 = (uint32_t)((bad >> (cur_lp & 63)) & 1) | (uint32_t)((bad >> (lp1 & 63)) & 1) << 1;
    } else {  // (the other tile first, so that this wave's pages are at hand afterwards; none past the sequence)
      const int other = my_tile ? cur_lp : lp1;
      uint32_t b_other = 0, b_mine = 0;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int l = i ? lp : other;
        if (l >= k.s.np) continue;
        if ((l >> 6) != chunk) set_chunk(l >> 6);
        const uint32_t x = (uint32_t)((bad >> (l & 63)) & 1);
        if (i) b_mine = x;
        else b_other = x;
      }
      bad2 = my_tile ? b_other | b_mine << 1 : b_mine | b_other << 1;
    }
    bads |= bad2;
    if ((bad2 >> my_tile) & 1) k_rows = 0;  // (hot: K is loaded all the same, from page 0, and masked; V is not any more)
    if (decltype(hot)::value || k_rows > 0) {
      k_at = static_cast<const unsigned char*>(uniform_ptr(page_base(lp & 63) + tp * tile_bytes));
      if constexpr (T == kI8) k_slot = (int64_t)__builtin_amdgcn_readlane(pg_id, lp & 63) * 2 * a.page + tp * kTile;
    }
    cur_p += KG;
    cur_tp += 2 * KG;
    while (cur_tp >= tpp) cur_tp -= tpp, ++cur_lp;
  };

  unsigned char* const ring = smem + kg * C::GROUP;  // K slots, V slots, scales
  const uint32_t lds0 = lds_addr(ring) + my_tile * C::TILE;
  // A load instruction takes RPI rows of a plane: this lane a 16-byte chunk of one, from where the row's order puts it.
  // Instruction I's rows are I * RPI behind, which changes the order by the swizzle of I * RPI alone.
  const int ln_row = lane / C::NCH, ln_ch = lane % C::NCH;
  const uint32_t ln_k = (ln_ch ^ C::kswz(ln_row)) * 16, ln_v = (ln_ch ^ C::vswz(ln_row)) * 16;
  const uint32_t row_b = (uint32_t)row_bytes, ln_off = ln_row * row_b;
  typedef __attribute__((address_space(3))) axk_u32x4* LdsPut;
  struct Stream {  // where an iteration's loads of this wave come from and go to (K, V; WR = 4: the one it loads, in k)
    const unsigned char *k, *v;
    uint32_t lds_k, lds_v;
    int rows_k, rows_v;
  };
  const uint32_t vmask = my_plane ? 0xffffffffu : 0u;
  auto stream = [&](int ks, int vs) {  // the next K into slot ks, the V before it into slot vs
    const uint32_t lk = lds0 + ks * C::PLANE, lv = lds0 + (NS + vs) * C::PLANE;
    if constexpr (WR == 4) {
      const int rk = k_rows, rv = v_rows;
      const unsigned char *ka = k_at, *va = v_at + plane_bytes;
      return Stream{static_cast<const unsigned char*>(uniform_ptr(my_plane ? va : ka)), nullptr, my_plane ? lv : lk, 0u,
                    my_plane ? rv : rk, 0};
    }
    return Stream{k_at, static_cast<const unsigned char*>(uniform_ptr(v_at + plane_bytes)), lk, lv, k_rows, v_rows};
  };
  const uint32_t ln_one = WR == 4 && my_plane ? ln_v : ln_k;
  // load `index` (0 .. IPW - 1) of an iteration
  auto load_one = [&](auto index, const Stream& st) {
    constexpr int I0 = decltype(index)::value, I = I0 % C::IPP, R = I * C::RPI;
    constexpr uint32_t TK = C::kswz(R) * 16, TV = C::vswz(R) * 16;
    constexpr bool V = I0 >= C::IPP;  // (WR = 2: K first)
    const uint32_t at = (WR == 4 ? ln_one ^ (TK ^ (vmask & (TK ^ TV))) : V ? ln_v ^ TV : ln_k ^ TK) + ln_off + R * row_b;
    lds_dma16_su_cached<I * 1024>(V ? st.v : st.k, at, V ? st.lds_v : st.lds_k);
  };
  // ... where a row has no token: zeros in its place (weight 0 times whatever lay there could be NaN)
  auto load_part = [&](auto index, const Stream& st) {
    constexpr int I0 = decltype(index)::value, I = I0 % C::IPP, R = I * C::RPI;
    constexpr bool V = I0 >= C::IPP;
    const int rows_in = V ? st.rows_v : st.rows_k;
    if (R + ln_row < rows_in) load_one(index, st);
    else *(LdsPut)(uintptr_t)((V ? st.lds_v : st.lds_k) + I * 1024 + lane * 16) = axk_u32x4{0u, 0u, 0u, 0u};
  };
  auto whole = [&](const Stream& st) { return st.rows_k == kTile && (WR == 4 || st.rows_v == kTile); };
  // int8: the scales of step i's pair, of this wave's tile: [tile][K, V][16]
  auto load_scales = [&](int i) {
    if constexpr (T == kI8) {
      const int row = l16 < k_rows ? l16 : 0;  // (past the last token its scale again: those scores are masked, weights zero)
      const int64_t at = (k_slot + row + (lane & 16 ? a.page : 0)) * a.hkv + kvh;
      if (lane < 32) lds_dma2(a.scales + at, lds_addr(ring) + 2 * NS * C::PLANE + (i & 7) * 256 + my_tile * 128);
    }
  };
  // ... read back: element e of group g for this lane's tokens 8 g + 4 h + e
  auto scales_of = [&](int i, int v, int g) {
    return *reinterpret_cast<const axk_u32x4*>(ring + 2 * NS * C::PLANE + (i & 7) * 256 + (g >> 1) * 128 + v * 64 +
                                               (8 * (g & 1) + 4 * h) * 4);
  };

  axk_f32x16 o[RT][DT];
  float m_run[RT], l_run[RT];  // l_run: this lane's half of the tokens
  float s[RT][16];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m_run[t] = -INFINITY, l_run[t] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][d][i] = 0.f;
  }
  const axk_f32x16 zero16 = {};

  // LDS addresses in bytes: a fragment's chunk is an exclusive or with a constant, as rows are powers of two of bytes.
  typedef const __attribute__((address_space(3))) axk_u32x4* LdsVec;
  typedef __attribute__((address_space(3))) axk_s16x4* LdsTr16;
  typedef __attribute__((address_space(3))) axk_i32x2* LdsTr8;
  const uint32_t ring0 = lds_addr(ring);
  // K row l32 of a pair as the A operand of step ks (8-bit: of steps ks and ks + 1)
  const uint32_t k_lane = ring0 + (l32 >> 4) * C::TILE + l16 * C::RBY + ((h ^ C::kswz(l16)) * 16);
  auto k_read = [&](uint32_t kb, int ks) {  // kb: k_lane of the pair's slot
    return *(LdsVec)(uintptr_t)(kb ^ ((T == kBf16 ? 32 : 16) * ks));
  };
  // V^T tile j % DT of the pair's tile j / DT as the A operand; MFMA k index (h, e) is token 8 (e / 4) + 4 h + e % 4
  const int vrow = T == kBf16 ? 4 * h + (l16 >> 2) : 8 * (l16 >> 3) + 4 * h + ((l16 >> 1) & 3);
  const int vch = T == kBf16 ? 2 * ((lane >> 4) & 1) + ((l16 >> 1) & 1) : (lane >> 4) & 1;
  const uint32_t v_lane = ring0 + NS * C::PLANE + vrow * C::RBY + ((vch ^ C::vswz(vrow)) * 16) + 8 * (l16 & 1);
  auto v_read = [&](uint32_t vb, int j) {  // vb: v_lane of the pair's slot
    const uint32_t at = (vb ^ ((T == kBf16 ? 64 : 32) * (j % DT))) + (j / DT) * C::TILE;
    if constexpr (T == kBf16) {
      const axk_s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr16)(uintptr_t)at);
      const axk_s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr16)(uintptr_t)(at + 8 * C::RBY));  // (kept alike)
      return __builtin_bit_cast(axk_u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const axk_i32x2 v = __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsTr8)(uintptr_t)at);
      return axk_u32x4{(uint32_t)v[0], (uint32_t)v[1], 0u, 0u};
    }
  };
  auto v_frag = [&](const axk_u32x4& w) {
    if constexpr (T == kBf16) return __builtin_bit_cast(axk_bf16x8, w);
    else return bf16_of<T>(w[0], w[1], a.inv_scale);
  };

  // what row tile t's row sees of the 32 tokens from `tok` on: history, then the row's ancestors
  auto visible = [&](int t, int tok, uint32_t bad2) {
    const uint64_t anc = node[t] >= 0 ? s_anc[node[t]] : 0;
    const int off = tok - base;
    uint32_t vis;
    if (off <= -kPair) vis = 0xffffffffu;
    else if (off < 0) vis = (0xffffffffu >> (kPair + off)) | ((uint32_t)anc << -off);
    else vis = off < 64 ? (uint32_t)(anc >> off) : 0u;
    return vis & ((bad2 & 1) ? 0xffff0000u : 0xffffffffu) & ((bad2 & 2) ? 0x0000ffffu : 0xffffffffu);
  };
  auto scale_scores = [&](int i) {  // int8: the K rows' scales
    if constexpr (T == kI8) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const axk_u32x4 w = scales_of(i, 0, g);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < RT; ++t) s[t][4 * g + e] *= bf16_bits_to_f32(w[e]);
      }
    }
  };
  auto pin = [](axk_f32x16& x) {  // a result stays where it is written; large ones in AGPRs
    if constexpr (RT * D >= 256) asm volatile("" : "+a"(x));
    else asm volatile("" : "+v"(x));
  };
  constexpr float kSlack = 8.0f;  // the reference maximum follows the scores in steps of more than 2^8
  float top[RT];         // the scores' maxima
  bool higher = false;   // wave-uniform: one has outgrown its reference
  auto raise_max = [&]() {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const bool raise = top[t] > m_run[t] + kSlack;
      const float alpha = raise ? __builtin_amdgcn_exp2f(m_run[t] - top[t]) : 1.0f;
      if (raise) m_run[t] = top[t];
      l_run[t] *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) {  // (tile by tile: all at once they would push what the loop keeps out of its registers)
        axk_f32x16 x = o[t][d];
        asm volatile("" : "+v"(x));
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= alpha;
        asm volatile("" : "+v"(x));
        o[t][d] = x;
        pin(o[t][d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    higher = false;
  };
  // the scores of step i are in s: masked, and their maximum taken up
  auto masked_pair = [&](int i, uint32_t bad2) { return (p_beg + i * KG) * kPair + kPair > base || bad2; };
  auto mask_scores = [&](int i, uint32_t bad2) {
    const bool masked = masked_pair(i, bad2);
    if (masked) {
      const int tok = (p_beg + i * KG) * kPair;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const uint32_t vis = visible(t, tok, bad2) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((vis >> (8 * (e >> 2) + (e & 3))) & 1)) s[t][e] = -INFINITY;
      }
    }
    return masked;
  };
  auto finish_scores = [&](auto hot, int i, uint32_t bad2, float (&mx)[RT]) {  // mx: the maxima of s, if nothing changes them
    scale_scores(i);
    const bool masked = !decltype(hot)::value && mask_scores(i, bad2);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (masked || T == kI8) {
        mx[t] = s[t][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx[t] = fmaxf(mx[t], s[t][e]);
      }
      top[t] = xor32_max(mx[t]) * c;
      higher |= __builtin_amdgcn_ballot_w64(top[t] > m_run[t] + kSlack) != 0;
    }
  };
  constexpr int KSTEP = T == kBf16 ? 1 : 2;  // steps of a K read
  auto qk_step = [&](const axk_u32x4& w, int ks, axk_f32x16 (&sn)[RT]) {
    if constexpr (T == kBf16) {
#pragma unroll
      for (int t = 0; t < RT; ++t) sn[t] = mfma_bf16_32x32x16(__builtin_bit_cast(axk_bf16x8, w), qb[t][ks], sn[t]);
    } else {
      const axk_bf16x8 f0 = bf16_of<T>(w[0], w[1], a.inv_scale), f1 = bf16_of<T>(w[2], w[3], a.inv_scale);
#pragma unroll
      for (int t = 0; t < RT; ++t) sn[t] = mfma_bf16_32x32x16(f0, qb[t][ks], sn[t]);
#pragma unroll
      for (int t = 0; t < RT; ++t) sn[t] = mfma_bf16_32x32x16(f1, qb[t][ks + 1], sn[t]);
    }
  };

  if (wave == 0) {  // (a bad tree sets *status whatever piece sees it)
    const uint64_t anc = ancestors(parent, a.nodes, a.status);
    s_anc[lane] = base >= 0 ? anc : 0;
    if (lane == 0) *s_odd = 0;
  }
  // K of pair 0, then an iteration's loads NS - 2 times (K of pair j, V of the one before); step -1 scores pair 0
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[t][e] = -INFINITY;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qb[t][ks]));  // the compiler's wait for q stays ahead of the loads
  }
  const std::false_type any{};
  int full = 0;  // iterations' loads in a row, up to the latest, that were all issued: they may be counted
  if (steps > 0) {
    next_pair(any);
    const Stream st = stream(0, 0);
    if (WR == 2 || !my_plane) for_each_index<C::IPP>([&](auto i) { load_part(i, st); });
    load_scales(0);
#pragma unroll 1
    for (int j = 1; j < NS - 1; ++j) {
      if (j < steps) next_pair(any);
      else v_at = k_at, v_rows = k_rows, bads <<= 2;  // (NS - 1 shifts before pair 0 is masked, however few pairs there are)
      if (j > steps) continue;
      const Stream sj = stream(j, j - 1);  // (V of the last pair comes with its K again)
      full = whole(sj) ? full + 1 : 0;
      if (full) for_each_index<C::IPW>([&](auto i) { load_one(i, sj); });
      else for_each_index<C::IPW>([&](auto i) { load_part(i, sj); });
      load_scales(min(j, steps - 1));
    }
  }

  // K of pair i + 1 and V of pair i have landed for every wave, and pair i - 1 has been read
  auto arrive = [&](auto hot) {
    if (decltype(hot)::value || full >= NS - 2)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * (C::IPW + (T == kI8))) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
  };
  // K of pair ld and V of the one before it are loaded; `full` then says whether their instructions are left to be issued
  auto issue = [&](auto hot, int ld) {
    constexpr bool HOT = decltype(hot)::value;
    if (HOT || ld < steps) next_pair(hot);
    else v_at = k_at, v_rows = k_rows, bads <<= 2;
    const Stream st = stream(ld & (NS - 1), (ld - 1) & (NS - 1));
    if constexpr (HOT) {
      load_scales(ld);
      return st;
    }
    const bool loads = ld <= steps;
    full = loads && whole(st) ? full + 1 : 0;
    if (loads) {
      if (!full) for_each_index<C::IPW>([&](auto x) { load_part(x, st); });
      load_scales(min(ld, steps - 1));
    }
    return st;
  };
  // every wave meets this barrier where a pair of either group holds a node
  auto holds_nodes = [&](int i) { return T != kI8 && (k.j * k.size + (i + 1) * KG) * kPair > base; };
  arrive(any);
  if (steps > 0) {  // the scores of pair 0
    const Stream st = issue(any, NS - 1);
    if (full) for_each_index<C::IPW>([&](auto x) { load_one(x, st); });
    axk_f32x16 sn[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) sn[t] = zero16;
    axk_u32x4 kf[2] = {k_read(k_lane, 0), k_read(k_lane, KSTEP)};
#pragma unroll
    for (int ks = 0; ks < KS; ks += KSTEP) {
      qk_step(kf[ks / KSTEP % 2], ks, sn);
      if (ks + 2 * KSTEP < KS) kf[ks / KSTEP % 2] = k_read(k_lane, ks + 2 * KSTEP);
#pragma unroll
      for (int t = 0; t < RT; ++t) pin(sn[t]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[t][e] = sn[t][e];
        asm volatile("" : "+v"(s[t][e]));  // (else the loop would carry s in AGPRs)
      }
    scale_scores(0);
    mask_scores(0, (bads >> (2 * (NS - 1))) & 3);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float mx = s[t][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
      m_run[t] = xor32_max(mx) * c;
    }
  }
  // Step i: pair i is weighted, pair i + 1 scored. No path leads around the products, since O would be copied where it meets the
  // others. HOT: whole pairs of history inside the pool, loads, and a next pair to score.
  auto step = [&](auto hot, const int i) {
    constexpr bool HOT = decltype(hot)::value;
    arrive(hot);
    // V of nodes: infinities and NaN are taken out, since weight 0 times them would be NaN; the rows that see them get them at
    // the end.
    if (!HOT && holds_nodes(i)) {
      const uint32_t at = ring0 + (NS + (i & (NS - 1))) * C::PLANE + (wr * 64 + lane) * 16;
      bool odd = false;
#pragma unroll
      for (int x = 0; x < C::PLANE / (WR * 1024); ++x) {
        axk_u32x4 w = *(LdsVec)(uintptr_t)(at + x * WR * 1024);
        uint32_t out = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t drop = 0;
          if constexpr (T == kBf16) {
            drop = ((w[e] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w[e] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) drop |= ((w[e] >> (8 * y)) & 0x7f) == 0x7f ? 0xffu << (8 * y) : 0u;
          }
          out |= drop;
          w[e] &= ~drop;
        }
        if (out) *(LdsPut)(uintptr_t)(at + x * WR * 1024) = w;
        odd |= out != 0;
      }
      if (odd) *s_odd = 1;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
    }
    const bool more = HOT || i + 1 < steps;  // wave-uniform: a next pair to score
    const Stream st = issue(hot, i + NS);
    const bool staged = HOT || full > 0;
    const uint32_t bad_n = (bads >> (2 * (NS - 1))) & 3;
    const uint32_t kb = k_lane + ((i + 1) & (NS - 1)) * C::PLANE, vb = v_lane + (i & (NS - 1)) * C::PLANE;
    // One MFMA step a stage, with the LDS read of a later one, a share of the loads and of the vector work beside it: the
    // scores of pair i + 1 run while pair i's become probabilities, and their maxima are taken while pair i is weighted. The
    // compiler orders inside a stage only.
    constexpr int NST = KS / KSTEP, KA = NST >= 8 ? 4 : NST / 2, VA = DT >= 4 ? 4 : DT;
    axk_f32x16 sn[RT];
    axk_u32x4 vf[VA];
    float m_use[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m_use[t] = m_run[t] == -INFINITY ? 0.f : m_run[t];
      sn[t] = zero16;
    }
    auto probs = [&](int lo, int hi) {
#pragma unroll
      for (int e = lo; e < hi; ++e) {
        const int t = e / 16, x = e % 16;
        s[t][x] = __builtin_amdgcn_exp2f(fmaf(s[t][x], c, -m_use[t]));
        l_run[t] += s[t][x];
      }
    };
    if (more) {
      axk_u32x4 kf[KA];
#pragma unroll
      for (int x = 0; x < KA; ++x) kf[x] = k_read(kb, x * KSTEP);
      __builtin_amdgcn_sched_barrier(0);
      for_each_index<NST>([&](auto stage) {
        constexpr int I = decltype(stage)::value;
        qk_step(kf[I % KA], I * KSTEP, sn);
        if constexpr (I + KA < NST) kf[I % KA] = k_read(kb, (I + KA) * KSTEP);
        else if constexpr (I + KA - NST < VA) vf[I + KA - NST] = v_read(vb, I + KA - NST);
        if constexpr (I < C::IPW)
          if (staged) load_one(stage, st);
        probs(I * 16 * RT / NST, (I + 1) * 16 * RT / NST);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          asm volatile("" : "+v"(l_run[t]));  // the sums and products stay in this stage
          pin(sn[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
#pragma unroll
      for (int x = KA; x < VA; ++x) vf[x] = v_read(vb, x);
    } else {
      if (staged) for_each_index<C::IPW>([&](auto x) { load_one(x, st); });
      probs(0, 16 * RT);
#pragma unroll
      for (int x = 0; x < VA; ++x) vf[x] = v_read(vb, x);
    }
    axk_bf16x8 pf[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if constexpr (T == kI8) {  // the V rows' scales; what is not seen stays zero whatever they hold
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const axk_u32x4 w = scales_of(i, 1, g);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[t][4 * g + e] = !HOT && s[t][4 * g + e] == 0.f ? 0.f : s[t][4 * g + e] * bf16_bits_to_f32(w[e]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        axk_u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(s[t][8 * x + 2 * e], s[t][8 * x + 2 * e + 1]);
        pf[t][x] = __builtin_bit_cast(axk_bf16x8, w);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    float mx[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) mx[t] = -INFINITY;
    auto take_scores = [&](int lo, int hi) {
#pragma unroll
      for (int e = lo; e < hi; ++e) {
        const int t = e / 16, x = e % 16;
        s[t][x] = sn[t][x];
        asm volatile("" : "+v"(s[t][x]));  // one copy out of the accumulator
        mx[t] = fmaxf(mx[t], s[t][x]);
      }
    };
      constexpr int PV = 2 * DT;
      for_each_index<PV>([&](auto stage) {
        constexpr int J = decltype(stage)::value;
        const axk_bf16x8 w = v_frag(vf[J % VA]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          o[t][J % DT] = mfma_bf16_32x32x16(w, pf[t][J / DT], o[t][J % DT]);
          pin(o[t][J % DT]);
        }
        if constexpr (J + VA < PV) vf[J % VA] = v_read(vb, J + VA);
        // (after the last tile's first product: sn and O then share no register)
        if constexpr (J >= DT) take_scores((J - DT) * 16 * RT / DT, (J - DT + 1) * 16 * RT / DT);
        __builtin_amdgcn_sched_barrier(0);
      });
    if (more) finish_scores(hot, i + 1, bad_n, mx);
  };
  // steps whose pair lies wholly before token x; the last step that finds all it needs in the history
  auto whole_steps = [&](int x) { return max((max(x, 0) / kPair - p_beg + KG - 1) / KG, 0); };
  const int hot_end = min(steps - NS, min(whole_steps(k.s.len) - NS, whole_steps(base) - KG));
  for (int i = 0; i < steps;) {
    // (no load that the compiler counts is in this loop: its waits would be waits for the direct loads too; and no raise, whose
    // 16 DT RT products would take the loop's registers)
    while (!higher && i < hot_end && full >= NS - 2 && !(bads & ((4u << (2 * NS)) - 1)) && at_hand()) step(std::true_type{}, i++);
    if (!higher) step(any, i++);
    if (higher) raise_max();
  }
  for (int i = steps; i < all_steps; ++i) {  // (the other group has one more)
    arrive(any);
    if (holds_nodes(i)) __builtin_amdgcn_s_barrier();
  }

  bool live[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l_run[t] = xor32_sum(l_run[t]);
    live[t] = node[t] >= 0 && s_anc[max(node[t], 0)] != 0;
    if (__builtin_amdgcn_ballot_w64(!live[t])) {  // rows of no node may have attended the history: they get zeros
      if (!live[t]) m_run[t] = -INFINITY, l_run[t] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][d][i] = live[t] ? o[t][d][i] : 0.f;
    }
  }
  if constexpr (KG == 2) {  // the second group's results through LDS to the first's waves, which hold the same rows
    __syncthreads();
    float2* const s_ml = reinterpret_cast<float2*>(smem);                       // [WR][RT][32]
    axk_f32x4* const s_o = reinterpret_cast<axk_f32x4*>(smem + WR * RT * 256);  // [WR][RT * DT * 4][64]
    static_assert(WR * RT * (256 + DT * 4 * 64 * 16) == C::JOIN, "the join's LDS");
    if (kg == 1) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if (h == 0) s_ml[(wr * RT + t) * 32 + l32] = make_float2(m_run[t], l_run[t]);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            s_o[((wr * RT + t) * DT * 4 + d * 4 + g) * 64 + lane] =
                axk_f32x4{o[t][d][4 * g], o[t][d][4 * g + 1], o[t][d][4 * g + 2], o[t][d][4 * g + 3]};
      }
    }
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float2 ml = s_ml[(wr * RT + t) * 32 + l32];
      const float m = fmaxf(m_run[t], ml.x);
      const float f0 = m_run[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[t] - m);
      const float f1 = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);
      m_run[t] = m;
      l_run[t] = l_run[t] * f0 + ml.y * f1;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const axk_f32x4 x = s_o[((wr * RT + t) * DT * 4 + d * 4 + g) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][d][4 * g + e] = o[t][d][4 * g + e] * f0 + x[e] * f1;
        }
    }
  }

  const int64_t slot0 = ((int64_t)gi * a.nb + blk) * RB;  // of this piece's rows in the workspace
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (node[t] < 0) continue;
    if (k.ns > 1) {
      const int64_t slot = slot0 + 32 * (RT * wr + t) + l32;
      if (h == 0) a.ml[slot] = make_float2(m_run[t], l_run[t]);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<axk_f32x4*>(a.po + slot * D + 32 * d + 8 * g + 4 * h) =
              axk_f32x4{o[t][d][4 * g], o[t][d][4 * g + 1], o[t][d][4 * g + 2], o[t][d][4 * g + 3]};
      continue;
    }
    // lanes l and l + 32 exchange halves, so that each holds 8 columns of two: 16 i + 8 h of its row
    const float inv = l_run[t] > 0.f ? 1.0f / l_run[t] : 0.f;
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) {
      const auto& ot = o[t][i / 2];
      const int e = 8 * (i % 2);
      const auto w0 = __builtin_amdgcn_permlane32_swap(pack_bf16x2(ot[e] * inv, ot[e + 1] * inv),
                                                       pack_bf16x2(ot[e + 4] * inv, ot[e + 5] * inv), false, false);
      const auto w1 = __builtin_amdgcn_permlane32_swap(pack_bf16x2(ot[e + 2] * inv, ot[e + 3] * inv),
                                                       pack_bf16x2(ot[e + 6] * inv, ot[e + 7] * inv), false, false);
      *reinterpret_cast<axk_u32x4*>(a.out + qrow[t] * D + 16 * i + 8 * h) = axk_u32x4{w0[0], w1[0], w0[1], w1[1]};
    }
  }
  // What was taken out of V, added to the rows that see it (each lane to four of every eight channels of its rows; an infinity
  // under a score of -inf, too, counts as one and not as 0 times it). Whole pairs were looked through, from the first that holds a
  // node (KG = 2: of the two of its step).
  // s_odd was last written before the last step's barrier.
  if (T != kI8 && __builtin_expect(*s_odd != 0, 0)) {
    wait_vmcnt<0>();
    const int p0 = k.j * k.size, first = p0 + max((max(base, 0) / kPair - p0) / KG * KG, 0);
    for (int tok = first * kPair; tok < min(k.s.len, p_end * kPair); ++tok) {
      const int pid = a.indices[k.s.pb + tok / a.page];
      if (pid < 0 || pid >= a.num_pages) continue;
      const unsigned char* row = head0 + ((int64_t)pid * 2 * a.page + tok % a.page) * row_bytes + plane_bytes;
      const int rel = tok - base;
#pragma unroll 1
      for (int t = 0; t < RT; ++t) {
        const int r = blk * RB + 32 * (RT * wr + t) + l32, nd = r < rows ? r / group : 0;
        const uint64_t anc = r < rows ? s_anc[nd] : 0;
        if (!anc || (rel >= 0 && !((anc >> rel) & 1))) continue;
        const int64_t out0 = (((int64_t)k.b * a.nodes + nd) * a.hq + kvh * group + r - nd * group) * D;
        const int64_t po0 = (slot0 + 32 * (RT * wr + t) + l32) * D;
#pragma unroll 1
        for (int x = 0; x < D / 2; ++x) {
          const int ch = 8 * (x >> 2) + 4 * h + (x & 3);
          const float v = T == kBf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[ch])
                                     : (row[ch] & 0x7f) == 0x7f ? NAN : 0.f;
          if (fabsf(v) < INFINITY) continue;
          if (k.ns > 1) a.po[po0 + ch] += v;
          else a.out[out0 + ch] = (uint16_t)f32_to_bf16_bits(bf16_bits_to_f32(a.out[out0 + ch]) + v);
        }
      }
    }
  }
}

// The log-sum-exp merge of a row's pieces, one wave a row. Rows of a sequence with a single piece are written already.
template <int D>
__global__ __launch_bounds__(64 * kMergeRows) void paged_tree_merge_kernel(TreeArgs a, int rb, int kg) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * kMergeRows + (threadIdx.x >> 6);  // (b T + t) HQ + head
  if (id >= (int64_t)a.batch * a.nodes * a.hq) return;
  const int b = __builtin_amdgcn_readfirstlane((int)(id / (a.nodes * a.hq)));
  const int rest = __builtin_amdgcn_readfirstlane((int)(id - (int64_t)b * a.nodes * a.hq));
  const int t = rest / a.hq, head = rest - t * a.hq, group = a.hq / a.hkv, kvh = head / group;
  const int parent = lane < a.nodes ? a.parents[(int64_t)b * a.nodes + lane] : -2;
  const Piece k = find_piece(a, b, false, kg);
  if (k.ns <= 1) return;
  uint16_t* const out = a.out + id * D + lane * PER;
  const int r = t * group + head - kvh * group, blk = r / rb;
  float acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  float l = 0.f;
  if (blk * rb < node_count(parent) * group) {  // (else no piece of the row's block has written anything)
    const int64_t step = (int64_t)a.hkv * a.nb * rb;
    const int64_t slot = (((int64_t)k.first * a.hkv + kvh) * a.nb + blk) * rb + r - blk * rb;
    const int ns = min(k.ns, a.groups / a.hkv - k.first);
    float m = -INFINITY;
    for (int j0 = 0; j0 < ns; j0 += 64) m = fmaxf(m, j0 + lane < ns ? a.ml[slot + (j0 + lane) * step].x : -INFINITY);
    m = wave_max(m);
    for (int j0 = 0; j0 < ns; j0 += 64) {
      const float2 x = j0 + lane < ns ? a.ml[slot + (j0 + lane) * step] : make_float2(-INFINITY, 0.f);
      // (a maximum of -inf: no score, and a sum of 0, or none but NaN, and a sum that is one)
      const float w = x.x == -INFINITY ? x.y : __builtin_amdgcn_exp2f(x.x - m);
      l += wave_sum(x.y * w);
      const int here = min(64, ns - j0);
      for (int i0 = 0; i0 < here; i0 += 8) {  // eight pieces' loads in flight
        float v[8][PER];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < PER; ++e) v[i][e] = a.po[(slot + (j0 + min(i0 + i, here - 1)) * step) * D + lane * PER + e];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float wi = i0 + i < here ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w),
                                                                                             min(i0 + i, 63))) : 0.f;
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += i0 + i < here ? v[i][e] * wi : 0.f;  // (0 times a NaN is one)
        }
      }
    }
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) out[e] = (uint16_t)f32_to_bf16_bits(acc[e] * inv);
}

template <int D, int T, int RT, int WR>
int launch(const TreeArgs& a, hipStream_t st) {
  using C = TreeCfg<D, T, RT, WR>;
  if constexpr (C::LDS > 64 * 1024) {  // to be allowed once on each device
    static AxkOnce once[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return AXK_E_LAUNCH;
    if (const int e = axk_raise_lds(once[dev & 63], reinterpret_cast<const void*>(&paged_tree_kernel<D, T, RT, WR>), C::LDS))
      return e;
  }
  AXK_LAUNCH_GATE();
  const int64_t grid = 8 * (int64_t)a.nb * ((a.groups + 7) / 8);
  hipLaunchKernelGGL((paged_tree_kernel<D, T, RT, WR>), dim3((unsigned)grid), dim3(256), C::LDS, st, a);
  if (a.split) {
    const int64_t rows = (int64_t)a.batch * a.nodes * a.hq;
    hipLaunchKernelGGL((paged_tree_merge_kernel<D>), dim3((unsigned)((rows + kMergeRows - 1) / kMergeRows)),
                       dim3(64 * kMergeRows), 0, st, a, C::RB, C::KG);
  }
  return axk_launch_status();
}

// The variant by the rows of a workgroup.
template <int D, int T>
int launch_rows(const TreeArgs& a, int rb, hipStream_t st) {
  if (rb == 64) return launch<D, T, 1, 2>(a, st);
  if constexpr (D == 256) return launch<D, T, 1, 4>(a, st);
  else if constexpr (D == 128) return rb == 128 ? launch<D, T, 2, 2>(a, st) : launch<D, T, 2, 4>(a, st);
  else return launch<D, T, 2, 2>(a, st);
}
template <int T>
int launch_type(const TreeArgs& a, int d, int rb, hipStream_t st) {
  switch (d) {
    case 64: return launch_rows<64, T>(a, rb, st);
    case 128: return launch_rows<128, T>(a, rb, st);
    default: return launch_rows<256, T>(a, rb, st);
  }
}

__attribute__((visibility("hidden"))) int launch_bf16(const TreeArgs& a, int d, int rb, hipStream_t st);
__attribute__((visibility("hidden"))) int launch_fp8(const TreeArgs& a, int d, int rb, hipStream_t st);
__attribute__((visibility("hidden"))) int launch_i8(const TreeArgs& a, int d, int rb, hipStream_t st);

}  // namespace axk_tree
