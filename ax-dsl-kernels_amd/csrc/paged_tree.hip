// Drafted tokens over a paged KV cache: their rows appended with the position rotation applied on the way, and the attention
// of a tree of them (paged_tree.h).
#include "paged_tree.h"

namespace {

using axk_tree::kBf16;
using axk_tree::kFp8;
using axk_tree::kI8;
using axk_tree::kMaxNodes;
using axk_tree::kSplitBatch;

// ---- rows into the cache ----
struct RopeArgs {
  const uint16_t *q, *k, *v;             // rows ld apart, heads hd apart
  int64_t ldq, hdq, ldk, hdk, ldv, hdv;
  const float *q_norm, *k_norm;          // [D] or NULL
  const void *cos, *sin;                 // [table, rot / 2], bf16 or f32
  const int *positions, *loc;            // [rows] or NULL; [rows, 2]
  uint16_t* q_out;                       // [rows, HQ, D]
  unsigned char* cache;
  uint16_t* scales;
  int* status;
  int rows, hq, hkv, rot, page;
  int64_t table, num_pages;
  float kv_scale, eps;
};

// Eight channels of a row as floats.
AXK_DEV void load8(const uint16_t* p, float (&x)[8]) {
  const axk_u32x4 w = *reinterpret_cast<const axk_u32x4*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}
AXK_DEV void load8(const float* p, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const axk_f32x4 w = *reinterpret_cast<const axk_f32x4*>(p + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = w[e];
  }
}
AXK_DEV axk_u32x4 pack8(const float (&x)[8]) {
  return axk_u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

// Row r's heads: HQ of q (if given), HKV of k, HKV of v; D / 8 lanes a head, eight channels each. q and k are normalised
// (y = x rsqrt(mean x^2 + eps) w) and channel pairs (i, i + rot / 2), i < rot / 2, turned by the row's angle, all in fp32 and
// rounded once, to what is stored: bf16, E4M3 of y * kv_scale, or int8 codes of the row's scale. A lane of a turned chunk
// loads its partner chunk too, which costs a cached load and no exchange. One launch for what a norm, a rotation and a store do in
// three: 4096 rows of 32 + 8 + 8 heads of 128 in 22.6 us (FP8 25.4, INT8 23.2), 4.5 TB/s of the 103 MB that they cannot do without;
// 16 rows in 4.1 us (4.6, 4.2), a launch and two dependent loads.
template <int D, int T, typename TAB>
__global__ __launch_bounds__(256) void paged_kv_write_rope_kernel(RopeArgs a) {
  constexpr int LPH = D / 8;  // lanes of a head
  const int heads = a.hq + 2 * a.hkv;
  const unsigned unit = blockIdx.x * 256u + threadIdx.x, hr = unit / LPH;
  const int c = unit % LPH;
  if (hr >= (unsigned)a.rows * (unsigned)heads) return;  // whole heads: the lanes of one act together
  const int row = (int)(hr / (unsigned)heads), head = (int)(hr - (unsigned)row * (unsigned)heads);
  const int pos = a.positions ? a.positions[row] : row;
  const int page = a.loc[2 * row], slot = a.loc[2 * row + 1];
  const bool is_q = head < a.hq, is_v = head >= a.hq + a.hkv;
  if (pos == -1) return;  // no row
  const bool bad_pos = pos < 0 || pos >= a.table;
  const bool bad_loc = page != -1 && (page < 0 || page >= a.num_pages || slot < 0 || slot >= a.page);
  if ((bad_pos || bad_loc) && a.status && c == 0) *a.status = 1;
  if (bad_pos || (!is_q && (bad_loc || page == -1))) return;

  const int kvh = head - a.hq - (is_v ? a.hkv : 0);
  const uint16_t* src = is_q ? a.q + row * a.ldq + head * a.hdq : is_v ? a.v + row * a.ldv + kvh * a.hdv
                                                                    : a.k + row * a.ldk + kvh * a.hdk;
  float x[8];
  load8(src + 8 * c, x);
  if (!is_v) {
    const int half = a.rot >> 4;  // chunks of half the turned channels
    const bool turned = c < 2 * half, low = c < half;
    const int pc = low ? c + half : c - half;
    float y[8], cs[8], sn[8];
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (turned) {
      load8(src + 8 * pc, y);
      const int64_t at = (int64_t)pos * (a.rot >> 1) + 8 * (low ? c : pc);
      load8(static_cast<const TAB*>(a.cos) + at, cs);
      load8(static_cast<const TAB*>(a.sin) + at, sn);
    }
    if (w) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
      sum = group_sum<(LPH < 16 ? LPH : 16)>(sum);
      if constexpr (LPH == 32) sum = xor16_sum(sum);
      const float r = 1.0f / sqrtf(sum * (1.0f / D) + a.eps);
      float wx[8];
      load8(w + 8 * c, wx);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= r * wx[i];
      if (turned) {
        load8(w + 8 * pc, wx);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= r * wx[i];
      }
    }
    if (turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = low ? x[i] * cs[i] - y[i] * sn[i] : x[i] * cs[i] + y[i] * sn[i];
    }
  }
  if (is_q) {
    *reinterpret_cast<axk_u32x4*>(a.q_out + ((int64_t)row * a.hq + head) * D + 8 * c) = pack8(x);
    return;
  }
  const int64_t at = (((int64_t)page * 2 + is_v) * a.page + slot) * a.hkv + kvh;
  if constexpr (T == kBf16) {
    *reinterpret_cast<axk_u32x4*>(reinterpret_cast<uint16_t*>(a.cache) + at * D + 8 * c) = pack8(x);
  } else {
    uint32_t b[2] = {0u, 0u};
    if constexpr (T == kFp8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i / 4] |= f32_to_e4m3(x[i] * a.kv_scale) << (8 * (i % 4));
    } else {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, LPH));
      const float s = kv_i8_scale(m), r = round_bf16(1.0f / s);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i / 4] |= ((uint32_t)(int)kv_i8_code(x[i], r) & 0xffu) << (8 * (i % 4));
      if (c == 0) a.scales[at] = (uint16_t)f32_to_bf16_bits(s);
    }
    *reinterpret_cast<uint2*>(a.cache + at * D + 8 * c) = make_uint2(b[0], b[1]);
  }
}

template <int T, typename TAB>
void launch_rope(const RopeArgs& a, int d, int64_t grid, hipStream_t st) {
  const dim3 g((unsigned)grid), t(256);
  switch (d) {
    case 64: hipLaunchKernelGGL((paged_kv_write_rope_kernel<64, T, TAB>), g, t, 0, st, a); break;
    case 128: hipLaunchKernelGGL((paged_kv_write_rope_kernel<128, T, TAB>), g, t, 0, st, a); break;
    default: hipLaunchKernelGGL((paged_kv_write_rope_kernel<256, T, TAB>), g, t, 0, st, a); break;
  }
}

bool head_dim_ok(int64_t d) { return d == 64 || d == 128 || d == 256; }
bool page_ok(int64_t page) { return page >= 16 && page % 16 == 0 && page <= 4096; }

// Elements that rows x heads of a strided operand span, from its first.
size_t span_of(int64_t rows, int64_t heads, int64_t ld, int64_t hd, int64_t d) {
  return (size_t)((rows - 1) * ld + (heads - 1) * hd + d);
}

int write_rope(const uint16_t* q, int64_t ldq, int64_t hdq, const uint16_t* k, int64_t ldk, int64_t hdk, const uint16_t* v,
               int64_t ldv, int64_t hdv, const float* q_norm, const float* k_norm, const void* cos, const void* sin,
               int table_dtype, int64_t table_rows, const int32_t* positions, const int32_t* loc, uint16_t* q_out, void* cache,
               int type, float kv_scale, uint16_t* scales, int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t rot,
               int64_t page_size, int64_t num_pages, float eps, int32_t* status, axk_stream_t stream) {
  AXK_REQUIRE(k && v && cache && loc && (rot == 0 || (cos && sin)) && (scales || type != kI8), AXK_E_NULL);
  AXK_REQUIRE(hq == 0 ? !q && !q_out && !q_norm : q && q_out, AXK_E_NULL);
  AXK_REQUIRE(rows >= 0 && rows <= (1 << 24) && hq >= 0 && hq <= 4096 && hkv > 0 && hkv <= 4096 && head_dim_ok(d), AXK_E_SHAPE);
  AXK_REQUIRE(rot >= 0 && rot <= d && rot % 16 == 0, AXK_E_SHAPE);
  AXK_REQUIRE(page_size > 0 && page_size <= (1 << 24) && num_pages > 0 && num_pages <= 0x7fffffff, AXK_E_SHAPE);
  AXK_REQUIRE(rot == 0 || (table_rows > 0 && (positions || table_rows >= rows)), AXK_E_SHAPE);
  if (type < 0) return -type;
  AXK_REQUIRE(table_dtype == AXK_DT_BF16 || table_dtype == AXK_DT_F32, AXK_E_DTYPE);
  const int64_t lds[] = {ldk, hdk, ldv, hdv, hq ? ldq : 0, hq ? hdq : 0};
  for (const int64_t x : lds) {
    AXK_REQUIRE(x >= 0 && x <= ((int64_t)1 << 32), AXK_E_SHAPE);
    AXK_REQUIRE(x % 8 == 0, AXK_E_ALIGN);
  }
  AXK_REQUIRE(axk_aligned(q, 16) && axk_aligned(k, 16) && axk_aligned(v, 16) && axk_aligned(q_out, 16) && axk_aligned(cos, 16) &&
                  axk_aligned(sin, 16) && axk_aligned(q_norm, 16) && axk_aligned(k_norm, 16) && axk_aligned(cache, 16) &&
                  axk_aligned(scales, 2) && axk_aligned(loc, 4) && axk_aligned(positions, 4) && axk_aligned(status, 4),
              AXK_E_ALIGN);
  if (rows == 0) return AXK_OK;
  const int64_t grid = (rows * (hq + 2 * hkv) * (d / 8) + 255) / 256;
  AXK_REQUIRE(axk_launch_fits(grid), AXK_E_SHAPE);
  const size_t slots = (size_t)num_pages * page_size * 2 * hkv, tab = (size_t)table_rows * (rot / 2) *
                                                                     (table_dtype == AXK_DT_F32 ? 4 : 2);
  const AxkSpan writes[] = {{q_out, (size_t)rows * hq * d * 2}, {cache, slots * d * (type == kBf16 ? 2 : 1)}, {scales, slots * 2},
                            {status, 4}};
  const AxkSpan reads[] = {{q, q ? span_of(rows, hq, ldq, hdq, d) * 2 : 0}, {k, span_of(rows, hkv, ldk, hdk, d) * 2},
                           {v, span_of(rows, hkv, ldv, hdv, d) * 2}, {q_norm, (size_t)d * 4}, {k_norm, (size_t)d * 4},
                           {rot ? cos : nullptr, tab}, {rot ? sin : nullptr, tab}, {positions, (size_t)rows * 4},
                           {loc, (size_t)rows * 8}};
  AXK_REQUIRE(axk_disjoint(writes, reads), AXK_E_ALIAS);
  RopeArgs a;
  a.q = q, a.k = k, a.v = v;
  a.ldq = ldq, a.hdq = hdq, a.ldk = ldk, a.hdk = hdk, a.ldv = ldv, a.hdv = hdv;
  a.q_norm = q_norm, a.k_norm = k_norm;
  a.cos = cos, a.sin = sin;
  a.positions = positions, a.loc = loc;
  a.q_out = q_out;
  a.cache = static_cast<unsigned char*>(cache);
  a.scales = scales;
  a.status = status;
  a.rows = (int)rows, a.hq = (int)hq, a.hkv = (int)hkv, a.rot = (int)rot, a.page = (int)page_size;
  a.table = rot ? table_rows : (int64_t)1 << 31;  // nothing is looked up without a rotation
  a.num_pages = num_pages;
  a.kv_scale = kv_scale;
  a.eps = eps;
  AXK_LAUNCH_GATE();
  hipStream_t st = axk_stream(stream);
  const bool f32 = table_dtype == AXK_DT_F32;
  switch (type) {
    case kBf16: f32 ? launch_rope<kBf16, float>(a, (int)d, grid, st) : launch_rope<kBf16, uint16_t>(a, (int)d, grid, st); break;
    case kFp8: f32 ? launch_rope<kFp8, float>(a, (int)d, grid, st) : launch_rope<kFp8, uint16_t>(a, (int)d, grid, st); break;
    default: f32 ? launch_rope<kI8, float>(a, (int)d, grid, st) : launch_rope<kI8, uint16_t>(a, (int)d, grid, st); break;
  }
  return axk_launch_status();
}

// ---- the tree's attention: how it is cut, from what the host knows ----
// A piece's least pairs of tokens. Us with 8, 4 and 2, 16 heads of 256: one sequence of 600 tokens 20.6, 20.4 and 19.0; of 5003
// tokens 24.8, 24.6 and 28.1, where shorter pieces cost more in the merge than their loops save.
constexpr int kMinPiece = 4;
struct TreePlan {
  int rb, nb, den, split;
  int64_t groups;
  size_t ml, po;
};
size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

TreePlan tree_plan(int64_t batch, int64_t nodes, int64_t hq, int64_t hkv, int64_t d, int64_t max_pairs) {
  TreePlan p;
  const int64_t rows = nodes * (hq / hkv);
  // Rows of a workgroup: two waves of rows and two of tokens up to 64 rows, as many rows as the registers hold beyond. Us with the
  // rule and the other choice, 16 sequences of 8000 tokens: 64 rows of 128 channels (8 KV heads) with 64 and 128 115 and 124 (FP8
  // 69 and 115, INT8 90 and 150), of 256 channels (2 heads) 59 and 63 (FP8 49 and 62, INT8 61 and 88); 96 rows of 128 channels
  // (4 heads) with 128 and 256 75 and 106 (INT8 91 and 142). Beyond 128 rows, 8 sequences of 32768 tokens: of 128 channels with 256
  // and 128 160 rows 370 and 409, 256 rows 399 and 413, 1024 rows 364 and 369 (256 rows of 16 x 8000 135 and 132); 512 rows of 256
  // channels with 128 and 64 653 and 804. Blocks of 256 rows of 64 channels measured 494 against 511, too little for a variant.
  p.rb = rows <= 64 ? 64 : rows > 128 && d == 128 ? 256 : 128;
  const int64_t nb = (rows + p.rb - 1) / p.rb;
  p.nb = (int)nb;
  const int64_t slots = p.rb == 64 && d <= 128 ? 512 : 256;  // workgroups at once: one or two a CU
  const int64_t den = slots / (hkv * nb);
  p.den = (int)(den > 1 ? den : 1);
  p.split = p.den > 1 && max_pairs > kMinPiece && batch <= kSplitBatch;
  p.groups = (batch + (p.split ? p.den : 0)) * hkv;
  const size_t slot_rows = (size_t)p.groups * nb * p.rb;
  p.ml = p.split ? round256(slot_rows * sizeof(float2)) : 0;
  p.po = p.split ? slot_rows * d * sizeof(float) : 0;
  return p;
}

int check_tree(int64_t batch, int64_t nodes, int64_t hq, int64_t hkv, int64_t d) {
  AXK_REQUIRE(batch > 0 && batch <= (1 << 20) && nodes > 0 && nodes <= kMaxNodes, AXK_E_SHAPE);
  AXK_REQUIRE(hkv > 0 && hkv <= 4096 && hq > 0 && hq % hkv == 0 && hq / hkv <= 16 && head_dim_ok(d), AXK_E_SHAPE);
  return AXK_OK;
}

int tree_verify(const uint16_t* q, const void* cache, int type, float kv_scale, const uint16_t* scales, const int32_t* indptr,
                const int32_t* indices, const int32_t* last, const int32_t* parents, uint16_t* out, int64_t nnz, int64_t batch,
                int64_t nodes, int64_t hq, int64_t hkv, int64_t d, int64_t page, int64_t num_pages, float sm_scale,
                int32_t* status, void* workspace, size_t workspace_bytes, axk_stream_t stream) {
  AXK_REQUIRE(q && cache && indptr && (indices || nnz == 0) && last && parents && out && (scales || type != kI8), AXK_E_NULL);
  const int rc = check_tree(batch, nodes, hq, hkv, d);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(page_ok(page) && num_pages > 0 && num_pages <= 0x7fffffff && nnz >= 0 && nnz * page <= 0x7fffff00, AXK_E_SHAPE);
  if (type < 0) return -type;
  AXK_REQUIRE(axk_aligned(q, 16) && axk_aligned(cache, 16) && axk_aligned(out, 16) && axk_aligned(scales, 2) &&
                  axk_aligned(indptr, 4) && axk_aligned(indices, 4) && axk_aligned(last, 4) && axk_aligned(parents, 4) &&
                  axk_aligned(status, 4),
              AXK_E_ALIGN);
  const TreePlan p = tree_plan(batch, nodes, hq, hkv, d, (nnz * page + 31) / 32);
  // (a merge always fits: where a sequence may be cut, den > 1, so that it has at most 128 blocks of up to 256 rows, or 256 of 64,
  // in at most kSplitBatch sequences: 2^23 waves)
  AXK_REQUIRE(axk_launch_fits(p.nb * (p.groups + 7)), AXK_E_SHAPE);
  const size_t need = p.ml + p.po;
  AXK_REQUIRE(!need || (workspace && workspace_bytes >= need && axk_aligned(workspace, 256)), AXK_E_WORKSPACE);
  const size_t qb = (size_t)batch * nodes * hq * d * 2, slots = (size_t)num_pages * page * 2 * hkv;
  const AxkSpan writes[] = {{out, qb}, {workspace, need}, {status, 4}};
  const AxkSpan reads[] = {{q, qb}, {cache, slots * d * (type == kBf16 ? 2 : 1)}, {scales, slots * 2},
                           {indptr, (size_t)(batch + 1) * 4}, {indices, (size_t)nnz * 4}, {last, (size_t)batch * 4},
                           {parents, (size_t)batch * nodes * 4}};
  AXK_REQUIRE(axk_disjoint(writes, reads), AXK_E_ALIAS);
  axk_tree::TreeArgs a;
  a.q = q;
  a.cache = static_cast<const unsigned char*>(cache);
  a.scales = scales;
  a.indptr = indptr, a.indices = indices, a.last = last, a.parents = parents;
  a.out = out;
  a.ml = static_cast<float2*>(workspace);
  a.po = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + p.ml);
  a.status = status;
  a.batch = (int)batch, a.nodes = (int)nodes, a.hq = (int)hq, a.hkv = (int)hkv, a.page = (int)page, a.nnz = (int)nnz;
  a.nb = p.nb, a.den = p.den, a.min_piece = kMinPiece, a.groups = (int)p.groups, a.split = p.split;
  a.num_pages = num_pages;
  a.scale = sm_scale * axk_tree::kLog2e;
  a.inv_scale = type == kFp8 ? 1.0f / kv_scale : 1.0f;
  hipStream_t st = axk_stream(stream);
  return type == kBf16 ? axk_tree::launch_bf16(a, (int)d, p.rb, st)
         : type == kFp8 ? axk_tree::launch_fp8(a, (int)d, p.rb, st)
                        : axk_tree::launch_i8(a, (int)d, p.rb, st);
}

}  // namespace

extern "C" int axk_paged_kv_write_rope(const uint16_t* q, int64_t ldq, int64_t hdq, const uint16_t* k, int64_t ldk, int64_t hdk,
                                       const uint16_t* v, int64_t ldv, int64_t hdv, const float* q_norm, const float* k_norm,
                                       const void* cos, const void* sin, int table_dtype, int64_t table_rows,
                                       const int32_t* positions, const int32_t* cache_location, uint16_t* q_out, void* kv_cache,
                                       int kv_dtype, float kv_scale, int64_t rows, int64_t num_qo_heads, int64_t num_kv_heads,
                                       int64_t head_dim, int64_t rot, int64_t page_size, int64_t num_pages, float eps,
                                       int32_t* status, axk_stream_t stream) {
  return write_rope(q, ldq, hdq, k, ldk, hdk, v, ldv, hdv, q_norm, k_norm, cos, sin, table_dtype, table_rows, positions,
                    cache_location, q_out, kv_cache, axk_kv_type(kv_dtype, kv_scale), kv_scale, nullptr, rows, num_qo_heads,
                    num_kv_heads, head_dim, rot, page_size, num_pages, eps, status, stream);
}

extern "C" int axk_paged_kv_write_rope_i8(const uint16_t* q, int64_t ldq, int64_t hdq, const uint16_t* k, int64_t ldk,
                                          int64_t hdk, const uint16_t* v, int64_t ldv, int64_t hdv, const float* q_norm,
                                          const float* k_norm, const void* cos, const void* sin, int table_dtype,
                                          int64_t table_rows, const int32_t* positions, const int32_t* cache_location,
                                          uint16_t* q_out, int8_t* kv_cache, uint16_t* kv_scales, int64_t rows,
                                          int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int64_t rot,
                                          int64_t page_size, int64_t num_pages, float eps, int32_t* status,
                                          axk_stream_t stream) {
  return write_rope(q, ldq, hdq, k, ldk, hdk, v, ldv, hdv, q_norm, k_norm, cos, sin, table_dtype, table_rows, positions,
                    cache_location, q_out, kv_cache, kI8, 1.0f, kv_scales, rows, num_qo_heads, num_kv_heads, head_dim, rot,
                    page_size, num_pages, eps, status, stream);
}

extern "C" size_t axk_paged_tree_verify_workspace_size(int64_t batch, int64_t nodes, int64_t num_qo_heads, int64_t num_kv_heads,
                                                       int64_t head_dim) {
  if (check_tree(batch, nodes, num_qo_heads, num_kv_heads, head_dim) != AXK_OK) return 0;
  const TreePlan p = tree_plan(batch, nodes, num_qo_heads, num_kv_heads, head_dim, 0x7fffffff);
  return p.ml + p.po;
}

extern "C" int axk_paged_tree_verify(const uint16_t* q, const void* kv_cache, int kv_dtype, float kv_scale,
                                     const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len,
                                     const int32_t* parents, uint16_t* out, int64_t nnz, int64_t batch, int64_t nodes,
                                     int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                     int64_t num_pages, float sm_scale, int32_t* status, void* workspace,
                                     size_t workspace_bytes, axk_stream_t stream) {
  return tree_verify(q, kv_cache, axk_kv_type(kv_dtype, kv_scale), kv_scale, nullptr, indptr, indices, last_page_len, parents,
                     out, nnz, batch, nodes, num_qo_heads, num_kv_heads, head_dim, page_size, num_pages, sm_scale, status,
                     workspace, workspace_bytes, stream);
}

extern "C" int axk_paged_tree_verify_i8(const uint16_t* q, const int8_t* kv_cache, const uint16_t* kv_scales,
                                        const int32_t* indptr, const int32_t* indices, const int32_t* last_page_len,
                                        const int32_t* parents, uint16_t* out, int64_t nnz, int64_t batch, int64_t nodes,
                                        int64_t num_qo_heads, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                        int64_t num_pages, float sm_scale, int32_t* status, void* workspace,
                                        size_t workspace_bytes, axk_stream_t stream) {
  return tree_verify(q, kv_cache, kI8, 1.0f, kv_scales, indptr, indices, last_page_len, parents, out, nnz, batch, nodes,
                     num_qo_heads, num_kv_heads, head_dim, page_size, num_pages, sm_scale, status, workspace, workspace_bytes,
                     stream);
}
