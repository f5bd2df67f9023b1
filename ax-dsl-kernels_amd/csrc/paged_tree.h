// Attention of a tree of drafted tokens over a paged KV cache (paged_tree_*.hip instantiate it per stored type).
//
// The cache and page table are those of paged_attn.hip. A sequence's tree is parents[b, t], t < T <= 64: the node's parent (a
// node before it), -1 (the last token of the history) or -2 (no node). The n nodes' K / V are the last n cached tokens, node t
// at position len - n + t. For query head g of KV head h, with A(t) node t and its ancestors,
//   o_tg = sum_j p_j v_j,  p = softmax over {history} + A(t) of scale q_tg . k_j.
//
// The rows of one (sequence, KV head) are r = t G + g (G query heads a KV head): a workgroup takes 32 WR of them and a piece of
// the sequence's tokens, in pairs of 16-token tiles (a tile never leaves its page). Its four waves are WR row slices times
// KG = 4 / WR token groups; a group keeps its pair (K rows, then V rows, as bf16) in LDS and every wave computes
// S^T = K Q^T (32 tokens x its 32 rows) and O^T += V^T P^T over the whole head dim on 32x32x16 MFMA.
#pragma once
#include <math.h>

#include <type_traits>

#include "axk_common.h"
#include "axk_host.h"
#include "axk_tree_common.h"

namespace axk_tree {

typedef float axk_f32x16 __attribute__((ext_vector_type(16)));
typedef int axk_i32x4 __attribute__((ext_vector_type(4)));

enum { kBf16 = 0, kFp8 = 1, kI8 = 2 };  // stored as bf16, as E4M3 of x * kv_scale, as int8 codes with a bf16 scale per row
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

// Inclusive sum over the lanes of a wave.
AXK_DEV int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// How the batch is cut: every sequence into pieces of P pairs, P such that all pieces of all row blocks and KV heads fill the
// chip once (total / den pairs; a sequence's last piece is shorter, so there are at most den + batch pieces). Every wave of
// both launches derives the same cut from the page table: the total is a float sum in a fixed order.
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
  auto pairs_at = [&](int b0) { return b0 + lane < a.batch ? pairs_of(seq_from(lo, hi, tail, a.page, a.nnz)) : 0; };
  float total = 0.f;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    load(b0);
    total += wave_sum((float)pairs_at(b0));
  }
  Piece k;
  k.b = -1;
  k.size = 0x40000000;
  if (a.split) {
    const int p = max(a.min_piece, (int)(total / (float)a.den) + 1);
    k.size = (p + kg - 1) / kg * kg;
  }
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) load(b0);
    const int pairs = pairs_at(b0);
    // at least one piece, which writes the zeros of a sequence without tokens
    const int n = b0 + lane < a.batch ? max(1, (int)((unsigned)(pairs + k.size - 1) / (unsigned)k.size)) : 0;
    const int incl = wave_scan(n), excl = base + incl - n;
    const bool mine = by_piece ? n > 0 && want >= excl && want < excl + n : b0 + lane == want;
    const uint64_t hit = __ballot(mine);
    if (hit) {
      const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)hit) - 1);
      k.b = b0 + src;
      k.ns = __builtin_amdgcn_readlane(n, src);
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

template <int D>
struct TreeCfg {
  static constexpr int KS = D / 16;   // 16-deep MFMA steps of Q K^T
  static constexpr int DT = D / 32;   // 32-wide tiles of O
  static constexpr int RB = D * 2;    // bytes of a bf16 row
  static constexpr int NCH = RB / 16; // its 16-byte chunks
  static constexpr int PLANE = kPair * RB;
  static constexpr int BUF = 2 * PLANE + 2 * kPair * 4;  // K, V, and the int8 scales of both
  // Chunk c of K row r is kept at chunk c ^ (r mod 16) and of V row r at c ^ 4 (r mod 4), so that a K fragment read (32 rows,
  // one chunk each) and a transposing V read (4 rows, 64 bytes each) cover all LDS banks.
  static AXK_DEV int kswz(int r) { return r & (NCH < 16 ? NCH - 1 : 15); }
  static AXK_DEV int vswz(int r) { return 4 * (NCH < 16 ? ((r >> 1) & 1) : (r & 3)); }
  static constexpr int OLD = D + 4;   // floats of an O row in LDS
};

AXK_DEV axk_f32x16 mfma_bf16_32x32x16(axk_bf16x8 a, axk_bf16x8 b, axk_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 16 stored bytes as bf16 chunks: one (bf16) or two (8-bit; int8: the codes, exact in bf16).
template <int T>
AXK_DEV void as_bf16(const axk_u32x4 w, float inv_scale, axk_u32x4 (&out)[T == kBf16 ? 1 : 2]) {
  if constexpr (T == kBf16) {
    out[0] = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t x = w[i / 2];
      uint32_t r;
      if constexpr (T == kFp8)
        r = __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, inv_scale, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, inv_scale, false));
      else
        r = pack_bf16x2((float)(int8_t)(x >> (16 * (i & 1))), (float)(int8_t)(x >> (16 * (i & 1) + 8)));
      out[i / 4][i % 4] = r;
    }
  }
}

template <int D, int T, int WR>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_tree_kernel(TreeArgs a) {
  using C = TreeCfg<D>;
  constexpr int KG = 4 / WR, NT = 64 * WR, RB = 32 * WR;
  constexpr int CPU = T == kBf16 ? 1 : 2;           // bf16 chunks of a 16-byte load
  constexpr int LPR = C::NCH / CPU;                 // loads of a row
  constexpr int RPU = NT / LPR < kPair ? NT / LPR : kPair;  // rows of one load of all the group's threads
  constexpr int UNITS = kPair / RPU;                // loads a thread and plane
  constexpr int LOADERS = RPU * LPR;                // threads of the group that load (all but for 8-bit rows of 64 bytes)
  static_assert(NT % LPR == 0 && UNITS * RPU == kPair, "a pair divides over the group's threads");
  constexpr int SLOTS = WR == 1 ? 1 : 2;            // pairs of a group in LDS
  extern __shared__ __align__(16) unsigned char smem[];

  const int sl = blockIdx.x >> 3;
  const int gi = sl / a.nb * 8 + (blockIdx.x & 7), blk = sl % a.nb;
  if (gi >= a.groups) return;
  const int kvh = gi % a.hkv;
  const Piece k = find_piece(a, gi / a.hkv, true, KG);
  if (k.b < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / WR, wr = wave % WR, gt = threadIdx.x - kg * NT;
  const int l16 = lane & 15, l32 = lane & 31, h = lane >> 5;
  const int group = a.hq / a.hkv, rows = a.nodes * group;

  const int parent = lane < a.nodes ? a.parents[(int64_t)k.b * a.nodes + lane] : -2;
  const int n = node_count(parent);
  const int base = k.s.len - n;  // the first node's position
  if (base < 0 && a.status && threadIdx.x == 0) *a.status = 1;

  // this lane's row (lanes l and l + 32 share it)
  const int r = blk * RB + 32 * wr + l32;
  const bool inside = r < rows;
  const int node = inside ? r / group : 0;
  const int64_t qrow = ((int64_t)k.b * a.nodes + node) * a.hq + kvh * group + (inside ? r - node * group : 0);
  if (blk * RB >= n * group) {  // no node of this block is one
    if (k.ns == 1)
      for (int i = threadIdx.x; i < RB * C::NCH; i += 256) {
        const int rr = blk * RB + i / C::NCH;
        if (rr < rows) {
          const int t = rr / group;
          const int64_t at = (((int64_t)k.b * a.nodes + t) * a.hq + kvh * group + rr - t * group) * D + i % C::NCH * 8;
          *reinterpret_cast<axk_u32x4*>(a.out + at) = axk_u32x4{0u, 0u, 0u, 0u};
        }
      }
    return;
  }
  const uint64_t anc_lane = ancestors(parent, a.nodes, a.status);
  uint64_t anc = ((uint64_t)__shfl((uint32_t)(anc_lane >> 32), node) << 32) | __shfl((uint32_t)anc_lane, node);
  const bool live = inside && anc != 0 && base >= 0;

  // a negative scale moves into Q's signs and a zero scale into zero rows, so that scores keep their order
  const float c = a.scale == 0.f ? 1.0f : fabsf(a.scale);
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, keep = live && a.scale != 0.f ? 0xffffffffu : 0u;
  axk_bf16x8 qb[C::KS];
#pragma unroll
  for (int s = 0; s < C::KS; ++s) {
    axk_u32x4 w = *reinterpret_cast<const axk_u32x4*>(a.q + qrow * D + 16 * s + 8 * h);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (w[e] ^ flip) & keep;
    qb[s] = __builtin_bit_cast(axk_bf16x8, w);
  }

  // this group's pairs p_beg + kg, + KG, .. before p_end
  const int p_all = pairs_of(k.s);
  const int p_beg = k.j * k.size, p_end = min(p_all, p_beg + k.size);
  const int steps = (p_end - p_beg + KG - 1) / KG;
  const int tpp = a.page / kTile;
  const int64_t row_bytes = (int64_t)a.hkv * D * (T == kBf16 ? 2 : 1), plane_bytes = (int64_t)a.page * row_bytes;
  const unsigned char* const head0 = a.cache + (int64_t)kvh * D * (T == kBf16 ? 2 : 1);

  // page ids, 64 at a time: lane l holds that of the sequence's page 64 chunk + l
  int chunk = -1, ids = 0;
  auto page_id = [&](int lp) {
    if ((lp >> 6) != chunk) {
      chunk = lp >> 6;
      const int j = (chunk << 6) + lane;
      ids = j < k.s.np ? a.indices[k.s.pb + j] : 0;
    }
    return __builtin_amdgcn_readlane(ids, lp & 63);
  };
  // the next pair's tiles: page and tile within it
  int cur_lp = (2 * (p_beg + kg)) / tpp, cur_tp = 2 * (p_beg + kg) - cur_lp * tpp;

  struct Tile {
    const unsigned char* k;  // K of the tile's first token; V lies plane_bytes behind
    int64_t at;              // its token slot in the pool's plane 0
    int valid;               // tokens
  };
  auto tile_of = [&](int lp, int tp, int first_tok) {
    Tile t;
    const bool in = lp < k.s.np;
    const int pid = page_id(in ? lp : max(k.s.np - 1, 0));
    const bool bad = pid < 0 || pid >= a.num_pages;
    t.valid = in ? min(kTile, k.s.len - first_tok) : 0;
    if (bad && t.valid > 0) {
      if (a.status && lane == 0) *a.status = 1;
      t.valid = 0;
    }
    const int64_t page = bad ? 0 : pid;
    t.at = page * 2 * a.page + tp * kTile;
    t.k = static_cast<const unsigned char*>(uniform_ptr(head0 + t.at * row_bytes));
    return t;
  };

  axk_u32x4 kraw[UNITS], vraw[UNITS];
  uint32_t vis_tiles = 0;  // rows of the pair in flight that hold tokens
  uint16_t sraw[2];
  int tok0 = 0;  // first token of the pair in flight
  // loads of the group's next pair into registers; a row without a token is read as the tile's first one
  auto load_pair = [&](int p) {
    const int lp2 = cur_tp + 1 == tpp ? cur_lp + 1 : cur_lp, tp2 = cur_tp + 1 == tpp ? 0 : cur_tp + 1;
    tok0 = p * kPair;
    const Tile ta = tile_of(cur_lp, cur_tp, tok0), tb = tile_of(lp2, tp2, tok0 + kTile);
    cur_tp += 2 * KG;
    while (cur_tp >= tpp) cur_tp -= tpp, ++cur_lp;
    const uint32_t rows_a = ta.valid > 0 ? (1u << ta.valid) - 1 : 0, rows_b = tb.valid > 0 ? (1u << tb.valid) - 1 : 0;
    vis_tiles = (rows_a & 0xffffu) | (rows_b << 16);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int i = (LOADERS < NT ? gt % LOADERS : gt) + u * NT, row = i / LPR, ch = i % LPR;
      const bool second = row >= kTile;
      const int64_t off = ((vis_tiles >> row) & 1) ? (row & 15) * row_bytes : 0;
      const unsigned char* src = (second ? tb.k : ta.k) + off + ch * 16;
      kraw[u] = *reinterpret_cast<const axk_u32x4*>(src);
      vraw[u] = *reinterpret_cast<const axk_u32x4*>(src + plane_bytes);
    }
    if constexpr (T == kI8) {
      const int row = lane & 31;
      const bool second = row >= kTile;
      const int64_t at = ((second ? tb.at : ta.at) + (((vis_tiles >> row) & 1) ? (row & 15) : 0)) * a.hkv + kvh;
      sraw[0] = a.scales[at];
      sraw[1] = a.scales[at + (int64_t)a.page * a.hkv];
    }
  };
  // the pair in flight into the group's LDS slot; rows without a token are zero (weight 0 times any byte could be NaN)
  auto store_pair = [&](unsigned char* buf) {
    if (LOADERS == NT || gt < LOADERS)
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int i = gt + u * NT, row = i / LPR, ch = (i % LPR) * CPU;
      const uint32_t there = ((vis_tiles >> row) & 1) ? 0xffffffffu : 0u;
      axk_u32x4 kc[CPU], vc[CPU];
      as_bf16<T>(kraw[u], a.inv_scale, kc);
      as_bf16<T>(vraw[u], a.inv_scale, vc);
#pragma unroll
      for (int j = 0; j < CPU; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) kc[j][e] &= there, vc[j][e] &= there;
        *reinterpret_cast<axk_u32x4*>(buf + row * C::RB + (((ch + j) ^ C::kswz(row)) * 16)) = kc[j];
        *reinterpret_cast<axk_u32x4*>(buf + C::PLANE + row * C::RB + (((ch + j) ^ C::vswz(row)) * 16)) = vc[j];
      }
    }
    if constexpr (T == kI8) {
      if (gt < 64) {
        const int row = lane & 31;
        const float s = bf16_bits_to_f32(sraw[lane >> 5]);
        reinterpret_cast<float*>(buf + 2 * C::PLANE)[lane] = ((vis_tiles >> row) & 1) ? s : 0.f;
      }
    }
  };

  axk_f32x16 o[C::DT];
#pragma unroll
  for (int t = 0; t < C::DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;  // l_run: this lane's half of the tokens
  const int kaddr = l32 * C::RB;
  const int vrow = 4 * h + (l16 >> 2);
  constexpr float kSlack = 8.0f;  // the reference maximum follows the scores in steps of more than 2^8

  // MASKED: some row may not see some of the pair's tokens
  auto compute = [&](auto masked, const unsigned char* buf, int tok, uint32_t rows_in) {
    constexpr bool MASKED = decltype(masked)::value;
    axk_f32x16 sn = {};
#pragma unroll
    for (int s = 0; s < C::KS; ++s) {
      const axk_bf16x8 kf = *reinterpret_cast<const axk_bf16x8*>(buf + kaddr + (((2 * s + h) ^ C::kswz(l32)) * 16));
      sn = mfma_bf16_32x32x16(kf, qb[s], sn);
    }
    float s[16], sv[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = sn[i];
    if constexpr (T == kI8) {
      const float* sc = reinterpret_cast<const float*>(buf + 2 * C::PLANE);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const axk_f32x4 ks = *reinterpret_cast<const axk_f32x4*>(sc + 8 * i + 4 * h);
        const axk_f32x4 vs = *reinterpret_cast<const axk_f32x4*>(sc + kPair + 8 * i + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * i + e] *= ks[e], sv[4 * i + e] = vs[e];
      }
    }
    uint32_t vis = 0;  // what the row sees of the pair's tokens: history, then its ancestors
    if constexpr (MASKED) {
      const int off = tok - base;
      if (off <= -kPair) vis = 0xffffffffu;
      else if (off < 0) vis = (0xffffffffu >> (kPair + off)) | ((uint32_t)anc << -off);
      else vis = off < 64 ? (uint32_t)(anc >> off) : 0u;
      vis &= rows_in;
      const uint32_t mine = vis >> (4 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = (mine >> (8 * (i >> 2) + (i & 3))) & 1;
        s[i] = seen ? s[i] : -INFINITY;
        if constexpr (T == kI8) sv[i] = seen ? sv[i] : 0.f;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = xor32_max(mx) * c;
    const bool raise = mx > m_run + kSlack;
    if (__builtin_amdgcn_ballot_w64(raise)) {
      const float alpha = raise ? __builtin_amdgcn_exp2f(m_run - mx) : 1.0f;
      if (raise) m_run = mx;
      l_run *= alpha;
#pragma unroll
      for (int t = 0; t < C::DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    axk_bf16x8 pf[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -m_use));
      l_run += s[i];
      if constexpr (T == kI8) s[i] *= sv[i];
    }
#pragma unroll
    for (int ti = 0; ti < 2; ++ti) {
      axk_u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(s[8 * ti + 2 * i], s[8 * ti + 2 * i + 1]);
      pf[ti] = __builtin_bit_cast(axk_bf16x8, w);
    }
    uint32_t odd = 0;
    const unsigned char* vb = buf + C::PLANE + vrow * C::RB + 8 * (l16 & 1);
    const int vch = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
#pragma unroll
    for (int ti = 0; ti < 2; ++ti)
#pragma unroll
      for (int t = 0; t < C::DT; ++t) {
        const unsigned char* va = vb + ti * kTile * C::RB + (((4 * t + vch) ^ C::vswz(vrow)) * 16);
        const axk_s16x4 v0 = lds_read_tr16(va), v1 = lds_read_tr16(va + 8 * C::RB);
        axk_u32x4 vw = __builtin_bit_cast(axk_u32x4, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        if constexpr (MASKED && T != kI8) {  // infinities and NaN left out: weight 0 times them would be NaN
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t lo = (vw[e] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u;
            const uint32_t hi = (vw[e] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u;
            odd |= lo | hi;
            vw[e] &= ~(lo | hi);
          }
        }
        o[t] = mfma_bf16_32x32x16(__builtin_bit_cast(axk_bf16x8, vw), pf[ti], o[t]);
      }
    if constexpr (MASKED && T != kI8) {
      if (__builtin_amdgcn_ballot_w64(odd != 0)) {  // .. and added for the rows that do see them
        for (int j = 0; j < kPair; ++j) {
          const unsigned char* row = buf + C::PLANE + j * C::RB + 8 * h;
          const bool seen = (vis >> j) & 1;
#pragma unroll
          for (int i = 0; i < 4 * C::DT; ++i) {
            const uint2 w = *reinterpret_cast<const uint2*>(row + ((i ^ C::vswz(j)) * 16));
            const float x[4] = {__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                                __uint_as_float(w.y & 0xffff0000u)};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[i / 4][4 * (i % 4) + e] += seen && (__float_as_uint(x[e]) & 0x7f800000u) == 0x7f800000u ? x[e] : 0.f;
          }
        }
      }
    }
  };

  unsigned char* const mine = smem + kg * SLOTS * C::BUF;
  if (steps > 0) load_pair(p_beg + kg);  // (past p_end for a group without a pair: a tile without tokens)
  for (int i = 0; i < steps; ++i) {
    unsigned char* buf = mine + (i % SLOTS) * C::BUF;
    const int p = p_beg + kg + i * KG, tok = tok0;
    const uint32_t rows_in = p < p_end ? vis_tiles : 0u;
    store_pair(buf);
    if (i + 1 < steps) load_pair(p + KG);
    if constexpr (WR == 1) {
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
    if (p < p_end) {
      if (tok + kPair > base || rows_in != 0xffffffffu) compute(std::true_type{}, buf, tok, rows_in);
      else compute(std::false_type{}, buf, tok, rows_in);
    }
  }
  l_run = xor32_sum(l_run);
  if (__builtin_amdgcn_ballot_w64(!live)) {  // rows of no node have attended with zero queries: they get zeros
    if (!live) m_run = -INFINITY, l_run = 0.f;
#pragma unroll
    for (int t = 0; t < C::DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][i] = live ? o[t][i] : 0.f;
  }

  const int64_t slot0 = ((int64_t)(k.first + k.j) * a.hkv + kvh) * a.nb + blk;  // of this piece's rows in the workspace
  if constexpr (KG == 1) {
    if (!inside) return;
    if (k.ns > 1) {
      const int64_t slot = slot0 * RB + 32 * wr + l32;
      if (h == 0) a.ml[slot] = make_float2(m_run, l_run);
#pragma unroll
      for (int t = 0; t < C::DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(a.po + slot * D + 32 * t + 8 * i + 4 * h) =
              make_float4(o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]);
      return;
    }
    // lanes l and l + 32 exchange halves, so that each holds 8 columns of two: 32 t + 16 i + 8 h of its row
    const float inv = l_run > 0.f ? 1.0f / l_run : 0.f;
#pragma unroll
    for (int i = 0; i < 2 * C::DT; ++i) {
      const auto& ot = o[i / 2];
      const int e = 8 * (i % 2);
      const auto w0 = __builtin_amdgcn_permlane32_swap(pack_bf16x2(ot[e] * inv, ot[e + 1] * inv),
                                                       pack_bf16x2(ot[e + 4] * inv, ot[e + 5] * inv), false, false);
      const auto w1 = __builtin_amdgcn_permlane32_swap(pack_bf16x2(ot[e + 2] * inv, ot[e + 3] * inv),
                                                       pack_bf16x2(ot[e + 6] * inv, ot[e + 7] * inv), false, false);
      *reinterpret_cast<axk_u32x4*>(a.out + qrow * D + 16 * i + 8 * h) = axk_u32x4{w0[0], w1[0], w0[1], w1[1]};
    }
  } else {
    // the groups' outputs of each row joined in LDS: every wave against the row's common maximum, then summed
    __syncthreads();  // the pairs have been read
    float2* const s_ml = reinterpret_cast<float2*>(smem);                   // [KG][RB]
    float* const s_o = reinterpret_cast<float*>(smem + KG * RB * sizeof(float2));  // [KG][RB][OLD]
    const int lr = 32 * wr + l32;
    if (h == 0) s_ml[kg * RB + lr] = make_float2(m_run, l_run);
    __syncthreads();
    float m_all = -INFINITY;
#pragma unroll
    for (int g = 0; g < KG; ++g) m_all = fmaxf(m_all, s_ml[g * RB + lr].x);
    const float f = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_all);
#pragma unroll
    for (int t = 0; t < C::DT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<axk_f32x4*>(s_o + (kg * RB + lr) * C::OLD + 32 * t + 8 * i + 4 * h) =
            axk_f32x4{o[t][4 * i] * f, o[t][4 * i + 1] * f, o[t][4 * i + 2] * f, o[t][4 * i + 3] * f};
    __syncthreads();
    constexpr int VPR = D / 4;  // groups of four columns
    for (int i = threadIdx.x; i < RB * VPR; i += 256) {
      const int row = i / VPR, col = i % VPR * 4, rr = blk * RB + row;
      if (rr >= rows) break;
      axk_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int g = 0; g < KG; ++g) mm = fmaxf(mm, s_ml[g * RB + row].x);
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const float2 x = s_ml[g * RB + row];
        ll += x.x == -INFINITY ? 0.f : x.y * __builtin_amdgcn_exp2f(x.x - mm);
        const axk_f32x4 v = *reinterpret_cast<const axk_f32x4*>(s_o + (g * RB + row) * C::OLD + col);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
      }
      if (k.ns > 1) {
        const int64_t slot = slot0 * RB + row;
        if (col == 0) a.ml[slot] = make_float2(mm, ll);
        *reinterpret_cast<axk_f32x4*>(a.po + slot * D + col) = sum;
      } else {
        const float inv = ll > 0.f ? 1.0f / ll : 0.f;
        const int t = rr / group;
        const int64_t at = (((int64_t)k.b * a.nodes + t) * a.hq + kvh * group + rr - t * group) * D + col;
        *reinterpret_cast<uint2*>(a.out + at) = make_uint2(pack_bf16x2(sum[0] * inv, sum[1] * inv),
                                                           pack_bf16x2(sum[2] * inv, sum[3] * inv));
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
      const float w = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - m);
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
          for (int e = 0; e < PER; ++e) acc[e] += wi != 0.f ? v[i][e] * wi : 0.f;
        }
      }
    }
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) out[e] = (uint16_t)f32_to_bf16_bits(acc[e] * inv);
}

template <int D, int T, int WR>
int launch(const TreeArgs& a, hipStream_t st) {
  using C = TreeCfg<D>;
  constexpr int KG = 4 / WR, RB = 32 * WR, SLOTS = WR == 1 ? 1 : 2;
  constexpr size_t pairs = (size_t)KG * SLOTS * C::BUF;
  constexpr size_t join = KG > 1 ? (size_t)KG * RB * (sizeof(float2) + sizeof(float) * C::OLD) : 0;
  constexpr size_t lds = pairs > join ? pairs : join;
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  if constexpr (lds > 64 * 1024) {  // to be allowed once on each device
    static AxkOnce once[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return AXK_E_LAUNCH;
    if (const int e = axk_raise_lds(once[dev & 63], reinterpret_cast<const void*>(&paged_tree_kernel<D, T, WR>), lds)) return e;
  }
  AXK_LAUNCH_GATE();
  const int64_t grid = 8 * (int64_t)a.nb * ((a.groups + 7) / 8);
  hipLaunchKernelGGL((paged_tree_kernel<D, T, WR>), dim3((unsigned)grid), dim3(256), lds, st, a);
  if (a.split) {
    const int64_t rows = (int64_t)a.batch * a.nodes * a.hq;
    hipLaunchKernelGGL((paged_tree_merge_kernel<D>), dim3((unsigned)((rows + kMergeRows - 1) / kMergeRows)),
                       dim3(64 * kMergeRows), 0, st, a, RB, KG);
  }
  return axk_launch_status();
}

template <int T>
int launch_type(const TreeArgs& a, int d, int wr, hipStream_t st) {
  switch (d) {
    case 64: return wr == 1 ? launch<64, T, 1>(a, st) : wr == 2 ? launch<64, T, 2>(a, st) : launch<64, T, 4>(a, st);
    case 128: return wr == 1 ? launch<128, T, 1>(a, st) : wr == 2 ? launch<128, T, 2>(a, st) : launch<128, T, 4>(a, st);
    default: return wr == 1 ? launch<256, T, 1>(a, st) : wr == 2 ? launch<256, T, 2>(a, st) : launch<256, T, 4>(a, st);
  }
}

__attribute__((visibility("hidden"))) int launch_bf16(const TreeArgs& a, int d, int wr, hipStream_t st);
__attribute__((visibility("hidden"))) int launch_fp8(const TreeArgs& a, int d, int wr, hipStream_t st);
__attribute__((visibility("hidden"))) int launch_i8(const TreeArgs& a, int d, int wr, hipStream_t st);

}  // namespace axk_tree
