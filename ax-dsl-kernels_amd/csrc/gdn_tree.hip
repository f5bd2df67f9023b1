// Gated DeltaNet (GDN) over a tree of drafted tokens, for gfx950: every branch's outputs from one read of the state, and the
// state after the branch that was accepted.
//
// Node t continues its parent's state (gdn.hip's step): S_t = e^{g_t} S_parent, u_t = beta_t (v_t - k_t^T S_t), S_t += k_t u_t^T,
// o_t = q_t^T S_t, with q, k, g and beta as there. Unrolled over A(t), node t and its ancestors, with G_t the sum of g over A(t):
//   S_t = e^{G_t} S_0 + sum_{i in A(t)} e^{G_t - G_i} k_i u_i^T
//   u_t = beta_t (v_t - e^{G_t} k_t^T S_0) - sum_{i in A(t) - t} beta_t e^{G_t - G_i} (k_t . k_i) u_i
//   o_t = e^{G_t} q_t^T S_0 + sum_{i in A(t)} e^{G_t - G_i} (q_t . k_i) u_i
// (a g whose e^g is zero is left out of the sums, and what came before it gets weight 0: axk_tree::forgets)
// so no node's state is ever formed: the verify kernel reads S_0 once, solves the unit lower triangular system for u and
// leaves u and g; the commit kernel applies the accepted node's branch to S_0.
#include "axk_host.h"
#include "axk_tree_common.h"

namespace {

using axk_tree::kMaxNodes;

constexpr int kD = 128;      // both head dims
constexpr int kCols = 32;    // state columns of a wave: two MFMA tiles, of its even and its odd columns

struct TreeGdn {
  const uint16_t *q, *k, *v, *a, *b;  // [B, T, NK, 128], [B, T, NV, 128], [B, T, NV]
  const float *a_log, *dt_bias;       // [NV]
  const float* state;                 // [B, NV, 128, 128]
  const int* parents;                 // [B, T]
  uint16_t* out;                      // [B, T, NV, 128]
  float* updates;                     // u
  float* gates;                       // g [B, T, NV]
  int* status;
  int nodes, nk, nv;
};

AXK_DEV axk_f32x4 mfma_f32_16x16x4(float a, float b, axk_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// x = hi + mid + lo with bf16 parts, to 2^-24 of x: a bf16 MFMA with each gives the fp32 product (the other operand is bf16).
AXK_DEV void split3(const float (&x)[8], axk_bf16x8& hi, axk_bf16x8& mid, axk_bf16x8& lo) {
  axk_u32x4 w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float p = x[2 * i], r = x[2 * i + 1];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const uint32_t u = pack_bf16x2(p, r);
      w[j][i] = u;
      p -= __uint_as_float(u << 16);
      r -= __uint_as_float(u & 0xffff0000u);
    }
  }
  hi = __builtin_bit_cast(axk_bf16x8, w[0]);
  mid = __builtin_bit_cast(axk_bf16x8, w[1]);
  lo = __builtin_bit_cast(axk_bf16x8, w[2]);
}

// TT 16-node tiles, W waves of 32 state columns each. Lane (l16, g) holds, as an MFMA operand's row, node 16 tt + l16; of a
// result, column l16 and rows 4 g + r. A result's register r is the right operand of the fp32 step over the rows 4 g + r, so
// u goes from one product into the next without leaving its registers.
//
// Bound by the state's bytes for many short trees (64 sequences x 8 nodes x 32 heads: 150 MB in 41.5 us, 3.6 TB/s; three waves a
// SIMD, since the rows of the inversion are read one ahead instead of all at once, against 50.1 us with two), by the chain from
// the state's arrival through the weights and the triangular solve to the outputs for wide ones (8 x 64 nodes 27 us, of which one
// sequence takes 24).
template <int TT, int W>
__global__ __launch_bounds__(64 * W, TT == 1 ? 3 : TT == 2 ? 2 : 1) void gdn_tree_verify_kernel(TreeGdn p) {
  constexpr int N = 16 * TT, LD = N + 4;
  __shared__ __align__(16) float s_a[N * LD];  // the system's lower part, its diagonal tiles inverted in place
  __shared__ __align__(16) float s_p[N * LD];  // the outputs' weights
  __shared__ double s_sum[N];                  // G
  __shared__ uint2 s_anc[N], s_kept[N];        // A(t), and those of it whose updates are left at t
  __shared__ float s_beta[N], s_rk[N], s_rq[N], s_dec[N];

  const int slices = kD / (kCols * W);
  const int slice = blockIdx.x % slices, bh = blockIdx.x / slices;
  const int b = bh / p.nv, hd = bh - b * p.nv, kh = hd / (p.nv / p.nk);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int col = (slice * W + wave) * kCols + 2 * l16;  // this lane's even column

  // the state's columns: rows 32 s + 8 g + j
  float2 st[4][8];
  const char* sp = reinterpret_cast<const char*>(p.state + (int64_t)bh * kD * kD);
  const uint32_t at0 = (8 * g * kD + col) * 4;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double w = __builtin_nontemporal_load(reinterpret_cast<const double*>(sp + (at0 + (32 * s + j) * kD * 4)));
      st[s][j] = __builtin_bit_cast(float2, w);
    }

  // the nodes' k and q rows as operands, zero past the last node
  axk_bf16x8 kf[TT][4], qf[TT][4];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const int t = 16 * tt + l16;
    const int64_t row = ((int64_t)b * p.nodes + min(t, p.nodes - 1)) * p.nk + kh;
    const uint32_t keep = t < p.nodes ? 0xffffffffu : 0u;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      axk_u32x4 x = *reinterpret_cast<const axk_u32x4*>(p.k + row * kD + 32 * s + 8 * g);
      axk_u32x4 y = *reinterpret_cast<const axk_u32x4*>(p.q + row * kD + 32 * s + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] &= keep, y[e] &= keep;
      kf[tt][s] = __builtin_bit_cast(axk_bf16x8, x);
      qf[tt][s] = __builtin_bit_cast(axk_bf16x8, y);
    }
  }

  // v of the nodes 4 g + r of every tile
  uint32_t vf[TT][4];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      vf[tt][r] = *reinterpret_cast<const uint32_t*>(
          p.v + (((int64_t)b * p.nodes + min(16 * tt + 4 * g + r, p.nodes - 1)) * p.nv + hd) * kD + col);

  // gates, and the tree (wave 0; lane t is node t)
  if (wave == 0) {
    const bool in = lane < p.nodes;
    const int64_t tok = (int64_t)b * p.nodes + min(lane, p.nodes - 1);
    const int parent = in ? p.parents[tok] : -2;
    const float x = bf16_bits_to_f32(p.a[tok * p.nv + hd]) + p.dt_bias[hd], be = bf16_bits_to_f32(p.b[tok * p.nv + hd]);
    const float gt = -expf(p.a_log[hd]) * (x > 20.0f ? x : log1pf(expf(x)));
    const uint64_t zero = __ballot(axk_tree::forgets(gt));
    double sum = axk_tree::forgets(gt) ? 0.0 : (double)gt;
    const uint64_t anc = axk_tree::ancestors_sum<true>(parent, p.nodes, slice == 0 && hd == 0 ? p.status : nullptr, sum);
    if (lane < N) {
      s_sum[lane] = sum;
      const uint64_t kept = anc & (~0ull << axk_tree::last_of(anc & zero));
      s_kept[lane] = make_uint2((uint32_t)kept, (uint32_t)(kept >> 32));
      s_anc[lane] = make_uint2((uint32_t)anc, (uint32_t)(anc >> 32));
      s_beta[lane] = 1.0f / (1.0f + expf(-be));
      s_dec[lane] = expf((float)sum) * (anc & zero ? 0.f : 1.0f);  // (0 times a NaN stays one, as in the recurrence)
    }
    if (in && slice == 0) p.gates[tok * p.nv + hd] = anc ? gt : 0.f;
  }
  // the norms: each lane sums a quarter of its row
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = (float)kf[tt][s][j], y = (float)qf[tt][s][j];
        kk = fmaf(x, x, kk);
        qq = fmaf(y, y, qq);
      }
    kk = xor32_sum(xor16_sum(kk));
    qq = xor32_sum(xor16_sum(qq));
    if (wave == 0 && g == 0) {
      s_rk[16 * tt + l16] = 1.0f / sqrtf(kk + 1e-6f);
      s_rq[16 * tt + l16] = 0.08838834764831845f / sqrtf(qq + 1e-6f);  // 128^-1/2
    }
  }
  __syncthreads();

  // Nodes whose key, step size or decay is not a number, and the branches behind them: nothing of theirs may meet another
  // branch, where weight 0 times it would be NaN. Their weights are zero and their results NaN.
  uint64_t lost;
  {
    const int t = min(lane, N - 1);
    const uint64_t anc = lane < N ? ((uint64_t)s_anc[t].y << 32) | s_anc[t].x : 0;
    const float all = s_rk[t] + s_beta[t] + s_dec[t];
    const uint64_t from = __ballot(anc != 0 && (!(fabsf(all) < INFINITY) || s_rk[t] == 0.f));
    lost = from ? __ballot((anc & from) != 0) : 0;
  }

  // the weights of node i (this lane's column of a product) for node t (its rows)
  for (int id = wave; id < TT * TT; id += W) {
    const int tt = id / TT, ii = id - tt * TT;
    if (ii > tt) continue;
    axk_f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < TT; ++x)
      if (x == tt)
#pragma unroll
        for (int y = 0; y < TT; ++y)
          if (y == ii)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              kk = mfma_bf16_16x16x32(kf[x][s], kf[y][s], kk);
              qk = mfma_bf16_16x16x32(qf[x][s], kf[y][s], qk);
            }
    const int i = 16 * ii + l16;
    const double si = s_sum[i];
    const float rk = s_rk[i];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * tt + 4 * g + r;
      const uint2 kept = s_kept[t];
      const bool sees = ((i < 32 ? kept.x >> i : kept.y >> (i - 32)) & 1) != 0 && !((lost >> t) & 1);  // (then i is not either)
      const float w = sees ? expf((float)(s_sum[t] - si)) * rk : 0.f;
      s_a[t * LD + i] = sees && i != t ? s_beta[t] * s_rk[t] * w * kk[r] : 0.f;
      s_p[t * LD + i] = sees ? s_rq[t] * w * qk[r] : 0.f;
    }
  }
  __syncthreads();
  // the diagonal tiles inverted: lane l16 solves for column l16 of (I + A)^-1, four lanes groups alike
  for (int tt = wave; tt < TT; tt += W) {
    float x[16];
    float* at = s_a + 16 * tt * LD + 16 * tt;
    axk_f32x4 row[2][4];  // a row ahead; all at once would take 120 registers, and occupancy with them
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (i + 1 < 16 && 4 * c <= i) row[(i + 1) & 1][c] = *reinterpret_cast<const axk_f32x4*>(at + (i + 1) * LD + 4 * c);
      float v = i == l16 ? 1.0f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) v = fmaf(-row[i & 1][j / 4][j % 4], x[j], v);
      x[i] = v;
      asm volatile("" : "+v"(x[i])::"memory");
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_wave_barrier();
    if (g == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) at[i * LD + l16] = x[i];
  }
  __syncthreads();

  // k^T S_0 and q^T S_0 of every node
  axk_f32x4 ks[TT][2], qs[TT][2];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int c = 0; c < 2; ++c) ks[tt][c] = qs[tt][c] = axk_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = c ? st[s][j].y : st[s][j].x;
      axk_bf16x8 part[3];
      split3(x, part[0], part[1], part[2]);
#pragma unroll
      for (int i = 2; i >= 0; --i)
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          ks[tt][c] = mfma_bf16_16x16x32(kf[tt][s], part[i], ks[tt][c]);
          qs[tt][c] = mfma_bf16_16x16x32(qf[tt][s], part[i], qs[tt][c]);
        }
      __builtin_amdgcn_sched_barrier(0);  // (one split at a time: their parts would take as many registers as the state)
    }

  // what is no number is taken out before a product that other nodes share and kept as the bits of its nodes, per column
  uint64_t taint[2] = {lost, lost};
  auto clean = [&](axk_f32x4 (&x)[2], int tt) {
    bool odd = false;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= !(fabsf(x[c][r]) < INFINITY);
    if (!__builtin_amdgcn_ballot_w64(odd)) return;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t bits = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!(fabsf(x[c][r]) < INFINITY)) bits |= 1u << (4 * g + r), x[c][r] = 0.f;
      bits |= __shfl_xor(bits, 16);
      bits |= __shfl_xor(bits, 32);
      taint[c] |= (uint64_t)bits << (16 * tt);
    }
  };
  axk_f32x4 u[TT][2];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    axk_f32x4 rhs[2], o[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * tt + 4 * g + r;
      const bool live = (s_anc[t].x | s_anc[t].y) != 0 && !((lost >> t) & 1);  // (no ancestors past the last node)
      const uint32_t vw = vf[tt][r];
      const float be = s_beta[t], dk = s_dec[t] * s_rk[t], dq = s_dec[t] * s_rq[t];
      rhs[0][r] = live ? be * (__uint_as_float(vw << 16) - dk * ks[tt][0][r]) : 0.f;
      rhs[1][r] = live ? be * (__uint_as_float(vw & 0xffff0000u) - dk * ks[tt][1][r]) : 0.f;
      o[0][r] = live ? dq * qs[tt][0][r] : 0.f;
      o[1][r] = live ? dq * qs[tt][1][r] : 0.f;
    }
#pragma unroll
    for (int ii = 0; ii < tt; ++ii) {
      const axk_f32x4 w = *reinterpret_cast<const axk_f32x4*>(s_a + (16 * tt + l16) * LD + 16 * ii + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c) rhs[c] = mfma_f32_16x16x4(-w[r], u[ii][c][r], rhs[c]);
    }
    clean(rhs, tt);
    {
      const axk_f32x4 w = *reinterpret_cast<const axk_f32x4*>(s_a + (16 * tt + l16) * LD + 16 * tt + 4 * g);
      u[tt][0] = u[tt][1] = axk_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c) u[tt][c] = mfma_f32_16x16x4(w[r], rhs[c][r], u[tt][c]);
    }
    clean(u[tt], tt);
#pragma unroll
    for (int ii = 0; ii <= tt; ++ii) {
      const axk_f32x4 w = *reinterpret_cast<const axk_f32x4*>(s_p + (16 * tt + l16) * LD + 16 * ii + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c) o[c] = mfma_f32_16x16x4(w[r], u[ii][c][r], o[c]);
    }
    axk_f32x4 u_out[2] = {u[tt][0], u[tt][1]};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * tt + 4 * g + r;
      if (t >= p.nodes) break;
      if (taint[0] | taint[1]) {
        const uint64_t anc = ((uint64_t)s_anc[t].y << 32) | s_anc[t].x;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (anc & taint[c]) o[c][r] = u_out[c][r] = NAN;
      }
      const int64_t at = (((int64_t)b * p.nodes + t) * p.nv + hd) * kD + col;
      *reinterpret_cast<uint32_t*>(p.out + at) = pack_bf16x2(o[0][r], o[1][r]);
      *reinterpret_cast<float2*>(p.updates + at) = make_float2(u_out[0][r], u_out[1][r]);
    }
  }
}

// The accepted branch applied to the state: S' = e^{G_n} S_0 + sum_{i in A(n)} e^{G_n - G_i} k_i u_i^T, each workgroup 32 rows
// of one head's state, each thread 4 of them x 4 columns. One read and one write of the state and the branch's rows of u bound it:
// 32 sequences x 32 heads in 24.4 us, 5.7 TB/s; a single sequence's 4 MB take 5.5 us, a launch's latency and two dependent loads.
struct TreeCommit {
  const float* state;
  const uint16_t* k;
  const float *updates, *gates;
  const int *parents, *accepted;
  float* out;
  int* status;
  int nodes, nk, nv;
};
constexpr int kRows = 32;

__global__ __launch_bounds__(256) void gdn_tree_commit_kernel(TreeCommit p) {
  __shared__ __align__(16) float s_k[kMaxNodes][kRows];  // the branch's weighted, normalised k of this workgroup's rows
  __shared__ int s_node[kMaxNodes];
  const int part = blockIdx.x & 3, bh = blockIdx.x >> 2;
  const int b = bh / p.nv, hd = bh - b * p.nv, kh = hd / (p.nv / p.nk);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c4 = (threadIdx.x & 31) * 4, r0 = threadIdx.x >> 5;  // rows r0 + 8 j

  const int64_t at0 = (int64_t)bh * kD * kD + (int64_t)part * kRows * kD + c4;
  axk_f32x4 s[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    s[j] = __builtin_nontemporal_load(reinterpret_cast<const axk_f32x4*>(p.state + at0 + (r0 + 8 * j) * kD));

  const bool in = lane < p.nodes;
  const int64_t tok = (int64_t)b * p.nodes + min(lane, p.nodes - 1);
  const int parent = in ? p.parents[tok] : -2;
  const int node = p.accepted[b];
  const float gt = in ? p.gates[tok * p.nv + hd] : 0.f;
  double sum = axk_tree::forgets(gt) ? 0.0 : (double)gt;
  const uint64_t anc = axk_tree::ancestors_sum<true>(parent, p.nodes, hd == 0 && part == 0 ? p.status : nullptr, sum);
  const int from = min(max(node, 0), kMaxNodes - 1);
  const uint64_t all = ((uint64_t)__shfl((uint32_t)(anc >> 32), from) << 32) | __shfl((uint32_t)anc, from);
  const uint64_t path = node >= 0 && node < p.nodes ? all : 0;
  if (node != -1 && path == 0 && p.status && threadIdx.x == 0) *p.status = 1;
  const double total = __shfl(sum, from);
  const int m = __builtin_popcountll(path);
  if (m == 0) {  // nothing accepted: the state as it was
    if (p.out != p.state)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        __builtin_nontemporal_store(s[j], reinterpret_cast<axk_f32x4*>(p.out + at0 + (r0 + 8 * j) * kD));
    return;
  }
  // the branch in order: its i-th node by wave i % 4, lanes two channels each
  const int rank = __builtin_popcountll(path & ((1ull << lane) - 1));
  const uint64_t zero = path & __ballot(axk_tree::forgets(gt));
  const float w = lane < axk_tree::last_of(zero) ? 0.f : expf((float)(total - sum));
  if (((path >> lane) & 1) && wave == 0) s_node[rank] = lane;
  for (int i = wave; i < m; i += 4) {
    const int t = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(((path >> lane) & 1) && rank == i)) - 1);
    const uint32_t x = *reinterpret_cast<const uint32_t*>(p.k + (((int64_t)b * p.nodes + t) * p.nk + kh) * kD + 2 * lane);
    const float x0 = __uint_as_float(x << 16), x1 = __uint_as_float(x & 0xffff0000u);
    const float rk = __shfl(w, t) / sqrtf(wave_sum(fmaf(x0, x0, x1 * x1)) + 1e-6f);
    if (lane >> 4 == part) {
      s_k[i][2 * (lane & 15)] = x0 * rk;
      s_k[i][2 * (lane & 15) + 1] = x1 * rk;
    }
  }
  __syncthreads();
  const float dec = expf((float)total) * (zero ? 0.f : 1.0f);
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[j][e] *= dec;
  for (int i = 0; i < m; ++i) {
    const int t = __builtin_amdgcn_readfirstlane(s_node[i]);
    const axk_f32x4 u = *reinterpret_cast<const axk_f32x4*>(p.updates + (((int64_t)b * p.nodes + t) * p.nv + hd) * kD + c4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float kv = s_k[i][r0 + 8 * j];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = fmaf(kv, u[e], s[j][e]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    __builtin_nontemporal_store(s[j], reinterpret_cast<axk_f32x4*>(p.out + at0 + (r0 + 8 * j) * kD));
}

int check(int64_t batch, int64_t nodes, int64_t nk, int64_t nv, int64_t dk, int64_t dv) {
  AXK_REQUIRE(batch > 0 && nodes > 0 && nodes <= kMaxNodes && nk > 0 && nv > 0 && nv % nk == 0, AXK_E_SHAPE);
  AXK_REQUIRE(dk == kD && dv == kD && nv <= 4096 && batch <= (1 << 20) && batch * nv <= (1 << 20), AXK_E_SHAPE);
  return AXK_OK;
}

template <int TT>
void launch_verify(const TreeGdn& p, int64_t heads, hipStream_t st) {
  // One wave a workgroup spreads few heads over the CUs, but every wave then works out the heads' weights alone. Us for W = 1 and
  // W = 4, at 32 heads a sequence: 8 nodes x 1 sequence 7.9 and 9.2, x 8 10.4 and 10.4, x 16 14.1 and 13.4; 32 nodes x 1 13.4 and
  // 13.0, x 8 18.3 and 15.0; 64 nodes x 1 29.8 and 24.4, x 8 39.5 and 27.0.
  if constexpr (TT == 1)
    if (heads <= 256) {
      hipLaunchKernelGGL((gdn_tree_verify_kernel<1, 1>), dim3((unsigned)(4 * heads)), dim3(64), 0, st, p);
      return;
    }
  hipLaunchKernelGGL((gdn_tree_verify_kernel<TT, 4>), dim3((unsigned)heads), dim3(256), 0, st, p);
}

}  // namespace

extern "C" int axk_gdn_tree_verify(const uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* a, const uint16_t* b,
                                   const float* a_log, const float* dt_bias, const float* state, const int32_t* parents,
                                   uint16_t* out, float* updates, float* gates, int64_t batch, int64_t nodes,
                                   int64_t num_k_heads, int64_t num_v_heads, int64_t head_k_dim, int64_t head_v_dim,
                                   int32_t* status, axk_stream_t stream) {
  AXK_REQUIRE(q && k && v && a && b && a_log && dt_bias && state && parents && out && updates && gates, AXK_E_NULL);
  const int rc = check(batch, nodes, num_k_heads, num_v_heads, head_k_dim, head_v_dim);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(axk_aligned(q, 16) && axk_aligned(k, 16) && axk_aligned(v, 4) && axk_aligned(a, 2) && axk_aligned(b, 2) &&
                  axk_aligned(a_log, 4) && axk_aligned(dt_bias, 4) && axk_aligned(state, 8) && axk_aligned(parents, 4) &&
                  axk_aligned(out, 4) && axk_aligned(updates, 8) && axk_aligned(gates, 4) && axk_aligned(status, 4),
              AXK_E_ALIGN);
  const size_t toks = (size_t)batch * nodes, vb = toks * num_v_heads * kD * 2, kb = toks * num_k_heads * kD * 2;
  const size_t gb = toks * num_v_heads * 2, hb = (size_t)num_v_heads * 4;
  const AxkSpan writes[] = {{out, vb}, {updates, 2 * vb}, {gates, 2 * gb}, {status, 4}};
  const AxkSpan reads[] = {{q, kb}, {k, kb}, {v, vb}, {a, gb}, {b, gb}, {a_log, hb}, {dt_bias, hb},
                           {state, (size_t)batch * num_v_heads * kD * kD * 4}, {parents, toks * 4}};
  AXK_REQUIRE(axk_disjoint(writes, reads), AXK_E_ALIAS);
  const TreeGdn p = {q, k, v, a, b, a_log, dt_bias, state, parents, out, updates, gates, status, (int)nodes, (int)num_k_heads,
                     (int)num_v_heads};
  AXK_LAUNCH_GATE();
  const int64_t heads = batch * num_v_heads;
  if (nodes <= 16) launch_verify<1>(p, heads, axk_stream(stream));
  else if (nodes <= 32) launch_verify<2>(p, heads, axk_stream(stream));
  else launch_verify<4>(p, heads, axk_stream(stream));
  return axk_launch_status();
}

extern "C" int axk_gdn_tree_commit(const float* state_in, const uint16_t* k, const float* updates, const float* gates,
                                   const int32_t* parents, const int32_t* accepted, float* state_out, int64_t batch,
                                   int64_t nodes, int64_t num_k_heads, int64_t num_v_heads, int64_t head_k_dim,
                                   int64_t head_v_dim, int32_t* status, axk_stream_t stream) {
  AXK_REQUIRE(state_in && k && updates && gates && parents && accepted && state_out, AXK_E_NULL);
  const int rc = check(batch, nodes, num_k_heads, num_v_heads, head_k_dim, head_v_dim);
  if (rc != AXK_OK) return rc;
  AXK_REQUIRE(axk_aligned(state_in, 16) && axk_aligned(state_out, 16) && axk_aligned(k, 4) && axk_aligned(updates, 16) &&
                  axk_aligned(gates, 4) && axk_aligned(parents, 4) && axk_aligned(accepted, 4) && axk_aligned(status, 4),
              AXK_E_ALIGN);
  const size_t toks = (size_t)batch * nodes, sb = (size_t)batch * num_v_heads * kD * kD * 4;
  const AxkSpan writes[] = {{state_out, sb}, {status, 4}};
  const AxkSpan reads[] = {{state_in == state_out ? nullptr : state_in, sb}, {k, toks * num_k_heads * kD * 2},
                           {updates, toks * num_v_heads * kD * 4}, {gates, toks * num_v_heads * 4}, {parents, toks * 4},
                           {accepted, (size_t)batch * 4}};
  AXK_REQUIRE(axk_disjoint(writes, reads), AXK_E_ALIAS);
  const TreeCommit p = {state_in, k, updates, gates, parents, accepted, state_out, status, (int)nodes, (int)num_k_heads,
                        (int)num_v_heads};
  AXK_LAUNCH_GATE();
  hipLaunchKernelGGL(gdn_tree_commit_kernel, dim3((unsigned)(4 * batch * num_v_heads)), dim3(256), 0, axk_stream(stream), p);
  return axk_launch_status();
}
