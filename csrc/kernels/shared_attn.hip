// Attention whose keys and values are shared, training forms (gfx950): forward, dQ and dK/dV passes of
//
//  * latent attention, expanded: per head h   k[t,h] = [k_nope[t,h] | k_rope[t]],  o = softmax(scale q k^T) v.
//    k_nope and v are the two halves of ONE up-projected row kv[t,h] (DA + DV wide); k_rope (DB wide) is one vector a
//    token, shared by the heads -- it is staged beside k_nope as a second LDS image and never copied per head;
//  * attention over a shared prefix: the B = G n sequences attend to the P prefix keys of their group g = b / n (no
//    mask, first plen[g] of them) and then causally to their own S keys (first len[b] of them):
//      o_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij)  over both ranges, one running softmax.
//
// Mathematics, all accumulation in fp32:
//   forward   S^T = K Q^T (query on the lane: row statistics are lane-local), P = exp2(S c - m), O^T += V^T P^T
//   backward  delta = rowsum(dO * O), P = exp(S - lse), dP = dO V^T, dS = P * (dP - delta),
//             dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO; dk_rope = sum over heads, d(prefix) = sum over the group's
//             rows -- fp32 partials summed in a fixed order, no atomics: bits do not depend on scheduling.
// P and dS are rounded to the 16-bit type before their products: they are matrix-instruction operands.
//
// Structure: waves of 32 query rows (forward, dQ) or 32 keys (dK/dV), tiles by LDS-DMA one tile ahead, XOR-swizzled
// images, transposed operands by ds_read_b64_tr_b16. A tile's descriptor covers exactly its valid rows, so rows past a
// length read as zero whatever memory holds there (a score is masked besides), and a tile's base is a 64-bit address:
// no offset of a long sequence passes 32 bits.
#include <torch/all.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <type_traits>
#include "dlgm_attn.h"
#include "dlgm_attn_host.h"

using namespace dlgm;

namespace {

constexpr int kBQ = 128;   // query rows of a forward / dQ workgroup, keys of a dK/dV workgroup
constexpr int kBKV = 64;   // keys of a forward / dQ tile
constexpr int kBQP = 32;   // queries of a dK/dV tile over a prefix ...
constexpr int kBQ2 = 64;   // ... and of latent attention
constexpr int kKvThreads = 512;

template <typename E>
struct SharedArgs {
  const E *q, *k, *v, *kr;  // kr: shared rope key [B, S, DB] (latent attention)
  const E *pk, *pv;         // prefix keys / values [G, P, Hkv, D]
  const E *o, *dout;        // backward: forward output (contiguous) and its gradient
  E* out;                   // forward output [B, S, Hq, DV]
  float* lse;               // [B, Hq, S]
  float* rows;              // backward [2, B, Hq, S]: -delta, then -lse / scale
  E* dq;                    // [B, S, Hq, DA + DB]
  E *dk, *dv, *dpk, *dpv;   // 16-bit gradients of k, v and the prefix (written directly where one part covers them)
  float *dk_part, *dv_part, *dpk_part, *dpv_part;  // fp32 partials
  float* dkr_part;          // [Hq, B, S, DB]
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, kr_sb, kr_ss;
  int64_t pk_sb, pk_ss, pk_sh, pv_sb, pv_ss, pv_sh, do_sb, do_ss, do_sh;
  int64_t dk_ss, dk_sh, dv_ss, dv_sh;  // row and head strides of dk and dv (batch stride: S rows)
  const int *lens, *plens;  // [B], [G] valid keys (null: all)
  int B, S, Hq, Hkv, P, n;  // n: sequences of a group (1 without a prefix)
  int nsplit;               // dK/dV of a prefix: parts the group's sequences are cut into
  int prefix_blocks;        // dK/dV workgroups that own prefix keys (they come first)
  float scale, scale_log2, neg_inv_scale;
  bool causal;

  // the length of b (g), in a scalar register
  __device__ __forceinline__ int len(int b) const { return lens ? clamp_len(lens[b], S) : S; }
  __device__ __forceinline__ int plen(int g) const { return plens ? clamp_len(plens[g], P) : P; }
};

// ---- forward: one workgroup per (b, q head, 128 queries). SPLIT 2: two waves to 32 queries, each taking every other tile,
// joined at the end -- for grids that leave a CU no second workgroup, whose only wave a SIMD then waits out every latency
// (3 x 777 ragged, 8 heads (128, 64, 128), 168 workgroups: 25.4 us with one, 22.3 with two; dQ 35.6 and 32.8).
template <typename E, int DA, int DB, int DV, bool PRE, int SPLIT>
__global__ __launch_bounds__(kThreads * SPLIT, 2) void shared_fwd_kernel(SharedArgs<E> p) {
  constexpr int KA = DA / 16, KB = DB / 16, KK = KA + KB, DT = DV / 32;
  constexpr int TA = kBKV * DA, TB = kBKV * DB, TV = kBKV * DV, SLOT = TA + TB + TV;
  constexpr int DBX = DB ? DB : 32;
  __shared__ __attribute__((aligned(16))) E smem[2 * SPLIT * SLOT];

  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = wid & 3, half = SPLIT > 1 ? wid >> 2 : 0;  // this wave's rows, and which tiles it takes
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int nqt = (p.S + kBQ - 1) / kBQ, group = p.Hq / p.Hkv;
  // the longest first, over all heads. Workgroups go to the XCDs in turn, so those of one (prefix group, kv head), which
  // read the same keys at about the same time, share an XCD where these are a multiple of 8. (Head by head on one XCD each,
  // two long ones met on every CU: 450 and 416 us at 2 x 4096 tokens, 32 heads (128, 64, 128), 82 and 71 at 2 x 2048, 16;
  // no gain from the XCD alone at 5 x 1300, 20 heads: 103 and 91.)
  const int per_kv = p.n * group, nbk = p.B / p.n * p.Hkv;
  const int bk = blockIdx.x % nbk, rem = blockIdx.x / nbk;
  const int qt = nqt - 1 - rem / per_kv, idx = rem % per_kv;
  const int grp = bk / p.Hkv, hk = bk % p.Hkv, hq = hk * group + idx % group, b = grp * p.n + idx / group;

  const int len = p.len(b);
  const int q0 = qt * kBQ, q0w = q0 + 32 * w, qcol = q0w + r;
  const E* qb = p.q + b * p.q_sb + hq * p.q_sh;
  const E* kb = p.k + b * p.k_sb + hk * p.k_sh;
  const E* vb = p.v + b * p.v_sb + hk * p.v_sh;
  const E* krb = DB ? p.kr + b * p.kr_sb : nullptr;
  const E* pkb = PRE ? p.pk + grp * p.pk_sb + hk * p.pk_sh : nullptr;
  const E* pvb = PRE ? p.pv + grp * p.pv_sb + hk * p.pv_sh : nullptr;
  const int plen = PRE ? p.plen(grp) : 0;
  const int np = (plen + kBKV - 1) / kBKV;
  const int kv_end = p.causal ? min(len, q0 + kBQ) : len;
  const int nt = q0 < len ? np + (kv_end + kBKV - 1) / kBKV : 0;  // queries past the length have no tile

  const RowTile<E, DA, kBKV, 0> ka(w, lane);
  const RowTile<E, DBX, kBKV, 0> kr(w, lane);
  const RowTile<E, DV, kBKV, 2> va(w, lane);
  auto stage = [&](int buf, int step) {
    const int t = step * SPLIT + half;
    if (SPLIT > 1 && t >= nt) return;
    E* img = smem + (buf * SPLIT + half) * SLOT;
    if (PRE && t < np) {
      const int row0 = t * kBKV;
      ka.issue(img, pkb + (int64_t)row0 * p.pk_ss, p.pk_ss, plen - row0, w);
      va.issue(img + TA + TB, pvb + (int64_t)row0 * p.pv_ss, p.pv_ss, plen - row0, w);
    } else {
      const int row0 = (t - np) * kBKV;
      ka.issue(img, kb + (int64_t)row0 * p.k_ss, p.k_ss, len - row0, w);
      if constexpr (DB > 0) kr.issue(img + TA, krb + (int64_t)row0 * p.kr_ss, p.kr_ss, len - row0, w);
      va.issue(img + TA + TB, vb + (int64_t)row0 * p.v_ss, p.v_ss, len - row0, w);
    }
  };

  if (nt > 0) stage(0, 0);  // on its way beside the q fragments
  vec8_t<E> qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qf[kk] = row8(qb + (int64_t)qcol * p.q_ss + 16 * kk + 8 * h, qcol < len);
  settle(qf);
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = (f32x16)(0.f);
  float m_run = -INFINITY, l_run = 0.f;
  RowFrag<DA, 0> kf(r, h);
  RowFrag<DBX, 0> krf(r, h);
  TrFrag<DV, 2> vf(h, i16, g4);

  // unrolled by two: the LDS buffer is a compile-time constant in each copy (immediate ds_read offsets)
  const int steps = (nt + SPLIT - 1) / SPLIT;
  auto tile = [&](auto bufc, int step) {
    constexpr int buf = decltype(bufc)::value;
    vm_drain();       // this tile's DMA has landed (this wave's pieces) ...
    __syncthreads();  // ... and every wave's; the other buffer's readers are done
    if (step + 1 < steps) stage(buf ^ 1, step + 1);
    const int t = step * SPLIT + half;
    if (SPLIT > 1 && t >= nt) return;
    const bool pre = PRE && t < np;
    const int kv0 = pre ? t * kBKV : (t - np) * kBKV, end = pre ? plen : len;
    const bool causal = p.causal && !pre;
    if (causal && kv0 > q0w + 31) return;  // whole tile above this wave's diagonal
    const E* ki = smem + (buf * SPLIT + half) * SLOT;
    const E* vi = ki + TA + TB;
    f32x16 s[2] = {(f32x16)(0.f), (f32x16)(0.f)};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const E* a = kk < KA ? ki + 32 * u * DA + kf(kk) : ki + TA + 32 * u * DB + krf(kk - KA);
        s[u] = mfma32(lds_read_b128(a), qf[kk], s[u]);
      }
    if (uniform((causal && kv0 + kBKV - 1 > q0w) || kv0 + kBKV > end)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int kv = kv0 + 32 * u + (i & 3) + 8 * (i >> 2) + 4 * h;
          if (kv >= end || (causal && kv > qcol)) s[u][i] = -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
    mx = fmaxf(mx, swap_halves(mx)) * p.scale_log2;
    if (__any(mx > m_run + kRescaleLog2)) {  // deferred rescale, wave-uniform
      const float m_new = fmaxf(m_run, mx);
      const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    vec8_t<E> pf[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = fast_exp2(s[u][i] * p.scale_log2 - m_use);
        s[u][i] = e;
        l_run += e;
      }
      pf[u][0] = pack8<E>(s[u], 0);
      pf[u][1] = pack8<E>(s[u], 8);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
          o[dt] = mfma32(vf.read(vi, dt, 32 * u + 16 * s2), pf[u][s2], o[dt]);
  };
  for (int t = 0; t < steps; t += 2) {
    tile(std::integral_constant<int, 0>{}, t);
    if (t + 1 < steps) tile(std::integral_constant<int, 1>{}, t + 1);
  }

  float l_tot = l_run + swap_halves(l_run);
  if constexpr (SPLIT > 1) {
    constexpr int LD = DV + 4;
    static_assert(sizeof(E) * 2 * SPLIT * SLOT >= 4 * kBQ * (LD + 2), "the second half's rows fit the tiles' space");
    float* row = reinterpret_cast<float*>(smem) + (32 * w + r) * LD;
    float* ml = reinterpret_cast<float*>(smem) + kBQ * LD + 2 * (32 * w + r);
    __syncthreads();  // every tile has been read
    if (half) {
      store_rows_f32<DT>(row, o, 1.f, h);
      if (h == 0) ml[0] = m_run, ml[1] = l_tot;
    }
    __syncthreads();
    if (half) return;
    const float m = fmaxf(m_run, ml[0]);
    const float f0 = l_tot == 0.f ? 0.f : fast_exp2(m_run - m), f1 = ml[1] == 0.f ? 0.f : fast_exp2(ml[0] - m);
    l_tot = l_tot * f0 + ml[1] * f1;
    m_run = m;
    add_rows_f32<DT>(row, o, f0, f1, h);
  }
  const bool some = qcol < len && l_tot != 0.f;  // a padded query row: zeros and -inf
  store_rows_bf16<DT>(p.out + (((int64_t)b * p.S + qcol) * p.Hq + hq) * DV, o, 1.f / l_tot, h, qcol < p.S, some);
  if (qcol < p.S && h == 0)
    p.lse[((int64_t)b * p.Hq + hq) * p.S + qcol] = some ? (m_run + log2f(l_tot)) * kLn2 : -INFINITY;
}

// ---- dQ: one workgroup per (b, q head, 128 queries), the forward's walk and split. It holds dO in registers, so it also
// forms delta and writes the [-delta, -lse/scale] rows the dK/dV pass starts its accumulators from (padded rows: 0, 0). delta
// is that of the output as stored, in 16 bits: the unrounded one would have to be kept in fp32 for every row.
template <typename E, int DA, int DB, int DV, bool PRE, int SPLIT>
__global__ __launch_bounds__(kThreads * SPLIT, 2) void shared_bwd_dq_kernel(SharedArgs<E> p) {
  constexpr int KA = DA / 16, KB = DB / 16, KK = KA + KB, KV = DV / 16, DT = (DA + DB) / 32;
  constexpr int TA = kBKV * DA, TB = kBKV * DB, TV = kBKV * DV, SLOT = TA + TB + TV;
  constexpr int DBX = DB ? DB : 32;
  __shared__ __attribute__((aligned(16))) E smem[2 * SPLIT * SLOT];

  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = wid & 3, half = SPLIT > 1 ? wid >> 2 : 0;  // this wave's rows, and which tiles it takes
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int nqt = (p.S + kBQ - 1) / kBQ, group = p.Hq / p.Hkv;
  const int per_kv = p.n * group, nbk = p.B / p.n * p.Hkv;
  const int bk = blockIdx.x % nbk, rem = blockIdx.x / nbk;
  const int qt = nqt - 1 - rem / per_kv, idx = rem % per_kv;
  const int grp = bk / p.Hkv, hk = bk % p.Hkv, hq = hk * group + idx % group, b = grp * p.n + idx / group;

  const int len = p.len(b);
  const int q0 = qt * kBQ, q0w = q0 + 32 * w, qcol = q0w + r;
  const bool in = qcol < len;
  const E* kb = p.k + b * p.k_sb + hk * p.k_sh;
  const E* vb = p.v + b * p.v_sb + hk * p.v_sh;
  const E* krb = DB ? p.kr + b * p.kr_sb : nullptr;
  const E* pkb = PRE ? p.pk + grp * p.pk_sb + hk * p.pk_sh : nullptr;
  const E* pvb = PRE ? p.pv + grp * p.pv_sb + hk * p.pv_sh : nullptr;
  const int plen = PRE ? p.plen(grp) : 0;
  const int np = (plen + kBKV - 1) / kBKV;
  const int kv_end = p.causal ? min(len, q0 + kBQ) : len;
  const int nt = q0 < len ? np + (kv_end + kBKV - 1) / kBKV : 0;

  const RowTile<E, DA, kBKV, 1> ka(w, lane);
  const RowTile<E, DBX, kBKV, 1> kr(w, lane);
  const RowTile<E, DV, kBKV, 0> va(w, lane);
  auto stage = [&](int buf, int step) {
    const int t = step * SPLIT + half;
    if (SPLIT > 1 && t >= nt) return;
    E* img = smem + (buf * SPLIT + half) * SLOT;
    if (PRE && t < np) {
      const int row0 = t * kBKV;
      ka.issue(img, pkb + (int64_t)row0 * p.pk_ss, p.pk_ss, plen - row0, w);
      va.issue(img + TA + TB, pvb + (int64_t)row0 * p.pv_ss, p.pv_ss, plen - row0, w);
    } else {
      const int row0 = (t - np) * kBKV;
      ka.issue(img, kb + (int64_t)row0 * p.k_ss, p.k_ss, len - row0, w);
      if constexpr (DB > 0) kr.issue(img + TA, krb + (int64_t)row0 * p.kr_ss, p.kr_ss, len - row0, w);
      va.issue(img + TA + TB, vb + (int64_t)row0 * p.v_ss, p.v_ss, len - row0, w);
    }
  };

  if (nt > 0) stage(0, 0);  // on its way beside the q and dO fragments
  const E* qb = p.q + b * p.q_sb + hq * p.q_sh + (int64_t)qcol * p.q_ss;
  const E* dob = p.dout + b * p.do_sb + hq * p.do_sh + (int64_t)qcol * p.do_ss;
  vec8_t<E> qf[KK], dof[KV];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qf[kk] = row8(qb + 16 * kk + 8 * h, in);
#pragma unroll
  for (int kk = 0; kk < KV; ++kk) dof[kk] = row8(dob + 16 * kk + 8 * h, in);
  float lse2 = INFINITY, nd = 0.f;
  {
    const int64_t rowc = ((int64_t)b * p.Hq + hq) * p.S + qcol;
    float acc = 0.f;
    if (in) {
      const E* orow = p.o + (((int64_t)b * p.S + qcol) * p.Hq + hq) * DV + 8 * h;
#pragma unroll
      for (int kk = 0; kk < KV; ++kk) {
        const vec8_t<E> ov = *reinterpret_cast<const vec8_t<E>*>(orow + 16 * kk);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc += (float)dof[kk][j] * (float)ov[j];
      }
      lse2 = p.lse[rowc] * kLog2e;
    }
    nd = -(acc + swap_halves(acc));
    if (qcol < p.S && h == 0 && half == 0) {
      p.rows[rowc] = nd;
      p.rows[(int64_t)p.B * p.Hq * p.S + rowc] = in ? p.lse[rowc] * p.neg_inv_scale : 0.f;
    }
  }
  settle(qf), settle(dof);
  f32x16 dqt[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dqt[dt] = (f32x16)(0.f);
  RowFrag<DA, 1> kf(r, h);
  RowFrag<DBX, 1> krf(r, h);
  RowFrag<DV, 0> vf(r, h);
  TrFrag<DA, 1> kt(h, i16, g4);
  TrFrag<DBX, 1> krt(h, i16, g4);

  const int steps = (nt + SPLIT - 1) / SPLIT;
  auto tile = [&](auto bufc, int step) {
    constexpr int buf = decltype(bufc)::value;
    vm_drain();
    __syncthreads();
    if (step + 1 < steps) stage(buf ^ 1, step + 1);
    const int t = step * SPLIT + half;
    if (SPLIT > 1 && t >= nt) return;
    const bool pre = PRE && t < np;
    const int kv0 = pre ? t * kBKV : (t - np) * kBKV, end = pre ? plen : len;
    const bool causal = p.causal && !pre;
    if (causal && kv0 > q0w + 31) return;
    const E* ki = smem + (buf * SPLIT + half) * SLOT;
    const E* vi = ki + TA + TB;
    const bool need_mask = uniform((causal && kv0 + kBKV - 1 > q0w) || kv0 + kBKV > end);
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // one 32-key half at a time: its scores and dP are 32 registers
      f32x16 s = (f32x16)(0.f), dp = (f32x16)(0.f);
      pin(kf.at), pin(vf.at), pin(kt.at);
      if constexpr (DB > 0) pin(krf.at), pin(krt.at);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const E* a = kk < KA ? ki + 32 * u * DA + kf(kk) : ki + TA + 32 * u * DB + krf(kk - KA);
        s = mfma32(lds_read_b128(a), qf[kk], s);
        if (kk < KV) dp = mfma32(lds_read_b128(vi + 32 * u * DV + vf(kk)), dof[kk], dp);
      }
      if (need_mask) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int kv = kv0 + 32 * u + (i & 3) + 8 * (i >> 2) + 4 * h;
          if (kv >= end || (causal && kv > qcol)) s[i] = -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fast_exp2(s[i] * p.scale_log2 - lse2) * (dp[i] + nd);
      const vec8_t<E> ds[2] = {pack8<E>(s, 0), pack8<E>(s, 8)};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
          const vec8_t<E> a = dt < DA / 32 ? kt.read(ki, dt, 32 * u + 16 * s2)
                                           : krt.read(ki + TA, dt - DA / 32, 32 * u + 16 * s2);
          dqt[dt] = mfma32(a, ds[s2], dqt[dt]);
        }
    }
  };
  for (int t = 0; t < steps; t += 2) {
    tile(std::integral_constant<int, 0>{}, t);
    if (t + 1 < steps) tile(std::integral_constant<int, 1>{}, t + 1);
  }
  if constexpr (SPLIT > 1) {
    constexpr int LD = DA + DB + 4;
    static_assert(sizeof(E) * 2 * SPLIT * SLOT >= 4 * kBQ * LD, "the second half's rows fit the tiles' space");
    float* row = reinterpret_cast<float*>(smem) + (32 * w + r) * LD;
    __syncthreads();  // every tile has been read
    if (half) store_rows_f32<DT>(row, dqt, 1.f, h);
    __syncthreads();
    if (half) return;
    add_rows_f32<DT>(row, dqt, 1.f, 1.f, h);
  }
  store_rows_bf16<DT>(p.dq + (((int64_t)b * p.S + qcol) * p.Hq + hq) * (DA + DB), dqt, p.scale, h, qcol < p.S, in);
}

// ---- dK / dV over a shared prefix: one workgroup per (128 keys, HP q heads of one kv head, a range of sequences). Keys
// of a sequence are seen by that sequence alone; keys of a prefix by the n sequences of its group, walked one after the
// other into the same accumulators (cut into nsplit parts where the prefix alone gives too few workgroups).
// A wave of 32 keys keeps K and the gradients in registers and V in LDS: two waves a SIMD. (The split of the latent kernel
// below, two waves to 32 keys, measured 1622 us here against 1306 at 8 x 1024 queries over 4096 + 1024 keys, 32/8 heads.)
template <typename E, int D, int HP>
__global__ __launch_bounds__(kThreads, 2) void prefix_bwd_dkdv_kernel(SharedArgs<E> p) {
  constexpr int KK = D / 16, DT = D / 32;
  constexpr int TA = kBQP * D, SLOT = 2 * TA;
  __shared__ __attribute__((aligned(16))) E smem[2 * SLOT + kBQ * D];
  __shared__ __attribute__((aligned(16))) float rc[2][64];  // [buf][-lse/scale 0..31 | -delta 32..63]
  E* vimg = smem + 2 * SLOT;

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int group = p.Hq / p.Hkv, nhp = p.Hq / HP;
  const bool pre = (int)blockIdx.x < p.prefix_blocks;
  int b0, b1, hq, k0, part = 0;  // sequences b0 .. b1, first head, first key
  if (pre) {
    const int work = xcd_remap(blockIdx.x, p.prefix_blocks);
    const int nkt = (p.P + kBQ - 1) / kBQ;
    k0 = work % nkt * kBQ;  // blocks of one (group, part, head pair) share their Q / dO stream
    int x = work / nkt;
    hq = x % nhp * HP;
    x /= nhp;
    part = x % p.nsplit;
    const int grp = x / p.nsplit;
    b0 = grp * p.n + (int)((int64_t)p.n * part / p.nsplit);
    b1 = grp * p.n + (int)((int64_t)p.n * (part + 1) / p.nsplit);
  } else {
    // the first keys first, over all heads (2 x 2048 tokens, 32/8 heads, the whole backward: 354 us head by head, 314 so)
    const int id = blockIdx.x - p.prefix_blocks, nbh = p.B * nhp;
    k0 = id / nbh * kBQ;
    hq = id % nbh % nhp * HP;
    b0 = id % nbh / nhp;
    b1 = b0 + 1;
  }
  const int hk = hq / group, hh = hq % group, grp = b0 / p.n;
  const int nkeys = pre ? p.plen(grp) : p.len(b0);
  const bool causal = p.causal && !pre;
  const int kw0 = k0 + 32 * w, key = kw0 + r;
  const int64_t k_ss = pre ? p.pk_ss : p.k_ss, v_ss = pre ? p.pv_ss : p.v_ss;
  const E* kb = pre ? p.pk + grp * p.pk_sb + hk * p.pk_sh : p.k + b0 * p.k_sb + hk * p.k_sh;
  const E* vb = pre ? p.pv + grp * p.pv_sb + hk * p.pv_sh : p.v + b0 * p.v_sb + hk * p.v_sh;

  // this wave's 32 keys stay in registers (B operand of S = Q K^T); the V rows go to LDS once
  vec8_t<E> kf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) kf[kk] = row8(kb + (int64_t)key * k_ss + 16 * kk + 8 * h, key < nkeys);
  settle(kf);
  const RowTile<E, D, kBQ, 0> vt(w, lane);
  vt.issue(vimg, vb + (int64_t)k0 * v_ss, v_ss, nkeys - k0, w);

  f32x16 dk[DT], dv[DT];  // dK^T, dV^T: [d][key]
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[dt] = (f32x16)(0.f), dv[dt] = (f32x16)(0.f);

  const RowFrag<D, 1> qf(r, h);
  const RowFrag<D, 0> vf(r, h);
  const TrFrag<D, 1> qt(h, i16, g4);
  const RowTile<E, D, kBQP, 1> qd(w, lane);  // of Q and of dO
  const int64_t nrow = (int64_t)p.B * p.Hq * p.S;
  // the walk: sequence, head of the pair, 32-query tile (from the diagonal on under the causal mask)
  const int t0 = causal ? k0 / kBQP : 0;
  struct Cursor {
    int b, hp, t, nt, len;
  };
  auto seek = [&](Cursor& c) {  // the first position at or behind c that has a tile
    while (c.t >= c.nt) {
      c.t = t0;
      if (c.b >= 0 && ++c.hp < HP && t0 < c.nt) return true;
      c.hp = 0;
      c.b = c.b < 0 ? b0 : c.b + 1;
      if (c.b >= b1) return false;
      c.len = p.len(c.b);
      c.nt = (c.len + kBQP - 1) / kBQP;
    }
    return true;
  };
  auto stage = [&](int buf, const Cursor& c) {
    const int q0 = c.t * kBQP, hd = hq + c.hp;
    const E* qb = p.q + c.b * p.q_sb + hd * p.q_sh + (int64_t)q0 * p.q_ss;
    E* img = smem + buf * SLOT;
    qd.issue(img, qb, p.q_ss, c.len - q0, w);
    qd.issue(img + TA, p.dout + c.b * p.do_sb + hd * p.do_sh + (int64_t)q0 * p.do_ss, p.do_ss, c.len - q0, w);
    if (w == 0) {  // the rows' terms: lanes 0 .. 31 -lse/scale, 32 .. 63 -delta
      const float* rows = p.rows + ((int64_t)c.b * p.Hq + hd) * p.S + q0;
      const int bytes = 4 * (p.S - q0);
      if (lane < 32) dma4_async(rows + nrow, bytes, 4 * lane, lds_at(&rc[buf][0]));
      else dma4_async(rows, bytes, 4 * (lane - 32), lds_at(&rc[buf][0]));
    }
  };

  auto tile = [&](auto bufc, const Cursor& c, bool more, const Cursor& next) {
    constexpr int buf = decltype(bufc)::value;
    vm_drain();       // this tile's LDS-DMA has landed ...
    __syncthreads();  // ... for every wave, and the other buffer's readers are done
    if (more) stage(buf ^ 1, next);
    const int q0 = c.t * kBQP;
    if (causal && q0 + kBQP - 1 < kw0) return;
    const E* qi = smem + buf * SLOT;
    const E* di = qi + TA;
    f32x16 s, dp;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int qr_ = (i & 3) + 8 * (i >> 2) + 4 * h;
      s[i] = rc[buf][qr_];  // S - lse/scale  ->  P = exp2(that * scale * log2e)
      dp[i] = rc[buf][32 + qr_];
    }
    const E* vi = vimg + 32 * w * D;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      s = mfma32(lds_read_b128(qi + qf(kk)), kf[kk], s);
      dp = mfma32(lds_read_b128(di + qf(kk)), lds_read_b128(vi + vf(kk)), dp);
    }
    if (uniform((causal && q0 < kw0 + 31) || q0 + kBQP > c.len || kw0 + 32 > nkeys)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int q = q0 + (i & 3) + 8 * (i >> 2) + 4 * h;
        if (key >= nkeys || q >= c.len || (causal && key > q)) s[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float pv = fast_exp2(s[i] * p.scale_log2);
      s[i] = pv;
      dp[i] *= pv;
    }
    const vec8_t<E> pf[2] = {pack8<E>(s, 0), pack8<E>(s, 8)}, dsf[2] = {pack8<E>(dp, 0), pack8<E>(dp, 8)};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        dv[dt] = mfma32(qt.read(di, dt, 16 * s2), pf[s2], dv[dt]);
        dk[dt] = mfma32(qt.read(qi, dt, 16 * s2), dsf[s2], dk[dt]);
      }
  };
  int left = nkeys - key;  // > 0: this key exists; beside the tiles in a vector register, the scalar ones are spilled here
  pin(left);
  Cursor cur{-1, 0, 0, 0, 0};
  if (k0 < nkeys && seek(cur)) {
    stage(0, cur);
    bool more = true;
    while (more) {
      Cursor next = cur;
      ++next.t;
      more = seek(next);
      tile(std::integral_constant<int, 0>{}, cur, more, next);
      if (!more) break;
      cur = next;
      ++next.t;
      more = seek(next);
      tile(std::integral_constant<int, 1>{}, cur, more, next);
      cur = next;
    }
  }
  vm_drain();  // a workgroup without a tile still has its V rows in flight

  // rows of this block exist up to `rows`; keys past the length get zeros
  const int rows = pre ? p.P : p.S;
  const int nparts = (group / HP) * (pre ? p.nsplit : 1);
  const int slot = (pre ? part * (group / HP) : 0) + hh / HP;
  const int64_t base = (int64_t)(pre ? grp : b0) * rows + key;
  if (nparts == 1) {
    store_rows_bf16<DT>((pre ? p.dpk : p.dk) + (base * p.Hkv + hk) * D, dk, p.scale, h, key < rows, left > 0);
    store_rows_bf16<DT>((pre ? p.dpv : p.dv) + (base * p.Hkv + hk) * D, dv, 1.f, h, key < rows, left > 0);
  } else if (key < rows) {
    const int64_t all = (int64_t)(pre ? p.B / p.n : p.B) * rows;  // rows of a part
    const int64_t at = ((slot * all + base) * p.Hkv + hk) * D;
    store_rows_f32<DT>((pre ? p.dpk_part : p.dk_part) + at, dk, p.scale, h, left > 0);
    store_rows_f32<DT>((pre ? p.dpv_part : p.dv_part) + at, dv, 1.f, h, left > 0);
  }
}

// ---- dK / dV of latent attention: one workgroup per (b, head, 128 keys).
// K, V, dK and dV of 32 keys are 240 registers at head dims 192 / 128: too many for two waves a SIMD, and one alone hides
// none of its latencies (2120 us at S 8192, 32 heads). So two waves share 32 keys, and every SIMD runs one of each kind:
//   the first   S_i = Q K^T, P_i = exp, P_i to LDS (fp32)  |  dV += P_i^T dO_i
//   the second  dK += dS_{i-1}^T Q_{i-1}, dP_i = dO_i V^T  |  dS_i = P_i (dP_i - delta)
// with a barrier at | and one per tile of 64 queries: the exponentials of one run beside the products of the other.
template <typename E, int DA, int DB, int DV>
__global__ __launch_bounds__(kKvThreads, 2) void latent_bwd_dkdv_kernel(SharedArgs<E> p) {
  constexpr int KA = DA / 16, KB = DB / 16, KK = KA + KB, KV = DV / 16;
  constexpr int DTK = (DA + DB) / 32, DTA = DA / 32, DTV = DV / 32;
  constexpr int TA = kBQ2 * DA, TB = kBQ2 * DB, TO = kBQ2 * DV, SLOT = TA + TB + TO;
  __shared__ __attribute__((aligned(16))) E smem[3 * SLOT];
  __shared__ __attribute__((aligned(16))) float rc[3][2 * kBQ2];  // [buf][-lse/scale of the rows | -delta]
  __shared__ __attribute__((aligned(16))) float pbuf[4][2][1024];  // [32 keys][32 queries]: P in accumulator order

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  // the first keys, which most queries see, first, over all heads; blocks of one head share its Q / dO stream (3 x 1111
  // tokens, 16 heads, the whole backward: 157 us head by head, 134 so)
  const int bh = blockIdx.x % (p.B * p.Hq), k0 = blockIdx.x / (p.B * p.Hq) * kBQ, hd = bh % p.Hq, b = bh / p.Hq;
  const int len = p.len(b);
  const int kg = w & 3, kw0 = k0 + 32 * kg, key = kw0 + r;
  const RowTile<E, DA, kBQ2, 1, 8> qa(w, lane);
  const RowTile<E, DB, kBQ2, 1, 8> qr(w, lane);
  const RowTile<E, DV, kBQ2, 1, 8> da(w, lane);
  const int64_t nrow = (int64_t)p.B * p.Hq * p.S;
  const int t0 = p.causal ? k0 / kBQ2 : 0, nt = k0 < len ? (len + kBQ2 - 1) / kBQ2 : 0;
  const E* qb = p.q + b * p.q_sb + hd * p.q_sh;
  const E* dob = p.dout + b * p.do_sb + hd * p.do_sh;
  const float* rowb = p.rows + (w == 0 ? nrow : 0) + ((int64_t)b * p.Hq + hd) * p.S;
  auto stage = [&](int buf, int t) {
    const int q0 = t * kBQ2;
    E* img = smem + buf * SLOT;
    qa.issue(img, qb + (int64_t)q0 * p.q_ss, p.q_ss, len - q0, w);
    qr.issue(img + TA, qb + (int64_t)q0 * p.q_ss + DA, p.q_ss, len - q0, w);
    da.issue(img + TA + TB, dob + (int64_t)q0 * p.do_ss, p.do_ss, len - q0, w);
    // the rows' terms (past the length 0, 0; those scores are masked)
    if (w < 2) dma4_async(rowb + q0, 4 * (p.S - q0), 4 * lane, lds_at(&rc[buf][w * kBQ2]));
  };
  // both kinds of wave take the same walk: at tile t, tiles t - 1 and t are in LDS while t + 1 arrives, three buffers.
  // first(buffer of t, of t - 1, t, whether t and t - 1 have work for these keys), second(buffer of t, whether)
  auto walk = [&](auto&& first, auto&& second) {
    if (t0 < nt) stage(0, t0);
    bool behind = false;
    int buf = 0, last = 2;
    for (int t = t0; t < nt; ++t) {
      vm_drain();
      __syncthreads();  // tile t has landed for every wave, and the buffer of tile t - 2 has no reader left
      const int free = 3 - buf - last;
      if (t + 1 < nt) stage(free, t + 1);
      const bool active = uniform(!(p.causal && t * kBQ2 + kBQ2 - 1 < kw0));
      first(buf, last, t, active, behind);
      __syncthreads();  // P of tile t is in LDS
      second(buf, active);
      behind = active;
      last = buf, buf = free;
    }
    first(buf, last, nt, false, behind);
  };

  // keys past the length get zeros
  const int64_t base = (int64_t)b * p.S + key;
  if (w < 4) {  // P and dV
    vec8_t<E> kf[KK];  // B operand of S = Q K^T
    const E* kb = p.k + b * p.k_sb + hd * p.k_sh + (int64_t)key * p.k_ss + 8 * h;
    const E* krb = p.kr + b * p.kr_sb + (int64_t)key * p.kr_ss + 8 * h;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) kf[kk] = row8(kk < KA ? kb + 16 * kk : krb + 16 * (kk - KA), key < len);
    settle(kf);
    f32x16 dv[DTV];  // dV^T: [d][key]
#pragma unroll
    for (int dt = 0; dt < DTV; ++dt) dv[dt] = (f32x16)(0.f);
    const RowFrag<DA, 1> qf0(r, h);
    const RowFrag<DB, 1> qrf0(r, h);
    const TrFrag<DV, 1> dt0(h, i16, g4);
    vec8_t<E> pf[2][2];
    walk(
        [&](int buf, int, int t, bool active, bool) {
          if (!active) return;
          const int q0 = t * kBQ2;
          RowFrag<DA, 1> qf = qf0;
          RowFrag<DB, 1> qrf = qrf0;
          qf.at += buf * SLOT, qrf.at += buf * SLOT + TA;
          f32x16 s[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[u][j] = rc[buf][32 * u + (j & 3) + 8 * (j >> 2) + 4 * h];  // S - lse/scale
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int u = 0; u < 2; ++u)
              s[u] = mfma32(lds_read_b128(smem + (kk < KA ? 32 * u * DA + qf(kk) : 32 * u * DB + qrf(kk - KA))), kf[kk], s[u]);
          if (uniform((p.causal && q0 < kw0 + 31) || q0 + kBQ2 > len || kw0 + 32 > len)) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int q = q0 + 32 * u + (j & 3) + 8 * (j >> 2) + 4 * h;
                if (key >= len || q >= len || (p.causal && key > q)) s[u][j] = -INFINITY;
              }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float* to = pbuf[kg][u] + 4 * lane;
#pragma unroll
            for (int j = 0; j < 16; ++j) s[u][j] = fast_exp2(s[u][j] * p.scale_log2);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<f32x4*>(to + 256 * j) = (f32x4){s[u][4 * j], s[u][4 * j + 1], s[u][4 * j + 2], s[u][4 * j + 3]};
            pf[u][0] = pack8<E>(s[u], 0), pf[u][1] = pack8<E>(s[u], 8);
          }
        },
        [&](int buf, bool active) {
          if (!active) return;
          TrFrag<DV, 1> dt_ = dt0;
          dt_.at += buf * SLOT + TA + TB;
#pragma unroll
          for (int dt = 0; dt < DTV; ++dt)
#pragma unroll
            for (int x = 0; x < 4; ++x) dv[dt] = mfma32(dt_.template read<E>(smem, dt, 16 * x), pf[x >> 1][x & 1], dv[dt]);
        });
    store_rows_bf16<DTV>(p.dv + base * p.dv_ss + hd * p.dv_sh, dv, 1.f, h, key < p.S, key < len);
  } else {  // dS and dK, one tile behind
    vec8_t<E> vf[KV];  // B operand of dP = dO V^T
    const E* vb = p.v + b * p.v_sb + hd * p.v_sh + (int64_t)key * p.v_ss + 8 * h;
#pragma unroll
    for (int kk = 0; kk < KV; ++kk) vf[kk] = row8(vb + 16 * kk, key < len);
    settle(vf);
    f32x16 dk[DTK];  // dK^T: [d][key]
#pragma unroll
    for (int dt = 0; dt < DTK; ++dt) dk[dt] = (f32x16)(0.f);
    const RowFrag<DV, 1> df0(r, h);
    const TrFrag<DA, 1> qt0(h, i16, g4);
    const TrFrag<DB, 1> qrt0(h, i16, g4);
    vec8_t<E> dsf[2][2];
    f32x16 dp[2];
    walk(
        [&](int buf, int last, int, bool active, bool behind) {
          if (behind) {
            TrFrag<DA, 1> qt = qt0;
            TrFrag<DB, 1> qrt = qrt0;
            qt.at += last * SLOT, qrt.at += last * SLOT + TA;
#pragma unroll
            for (int dt = 0; dt < DTK; ++dt)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                dk[dt] = mfma32(dt < DTA ? qt.template read<E>(smem, dt, 16 * x) : qrt.template read<E>(smem, dt - DTA, 16 * x),
                                dsf[x >> 1][x & 1], dk[dt]);
          }
          if (active) {
            RowFrag<DV, 1> df = df0;
            df.at += buf * SLOT + TA + TB;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < 16; ++j) dp[u][j] = rc[buf][kBQ2 + 32 * u + (j & 3) + 8 * (j >> 2) + 4 * h];  // dP - delta
#pragma unroll
            for (int kk = 0; kk < KV; ++kk)
#pragma unroll
              for (int u = 0; u < 2; ++u) dp[u] = mfma32(lds_read_b128(smem + 32 * u * DV + df(kk)), vf[kk], dp[u]);
          }
        },
        [&](int, bool active) {
          if (!active) return;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float* from = pbuf[kg][u] + 4 * lane;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const f32x4 pv = *reinterpret_cast<const f32x4*>(from + 256 * j);
#pragma unroll
              for (int x = 0; x < 4; ++x) dp[u][4 * j + x] *= pv[x];
            }
            dsf[u][0] = pack8<E>(dp[u], 0), dsf[u][1] = pack8<E>(dp[u], 8);
          }
        });
    // one head owns its k_nope rows, the rope part is summed over the heads
    store_rows_bf16<DTA>(p.dk + base * p.dk_ss + hd * p.dk_sh, *reinterpret_cast<f32x16(*)[DTA]>(dk), p.scale, h, key < p.S,
                         key < len);
    if (key < p.S)
      store_rows_f32<DB / 32>(p.dkr_part + (((int64_t)hd * p.B + b) * p.S + key) * DB, dk + DTA, p.scale, h, key < len);
  }
}

// Sum of the fp32 parts in a fixed order -> 16 bits: dk_rope, or up to four tensors of a prefix backward (grid.y)
template <typename E>
struct SumArgs {
  const float* part[4];
  E* out[4];
  int64_t n[4];
  int parts[4];
};
template <typename E>
__global__ __launch_bounds__(256) void sum_parts_kernel(SumArgs<E> a) {
  const int y = blockIdx.y;
  const float* part = a.part[y];
  const int64_t n = a.n[y];
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
    f32x8 s = (f32x8)(0.f);
    for (int k = 0; k < a.parts[y]; ++k) s += *reinterpret_cast<const f32x8*>(part + k * n + i);
    store8f(a.out[y] + i, s);
  }
}

// forward and dQ: two waves to 32 queries where the grid leaves every CU at most one workgroup; and where it leaves two to
// latent attention over long sequences, whose first and last tiles differ so much that the second 256 workgroups are better
// handed out as the first end (1 x 4096 tokens, 16 heads: forward 133 and 116 us, backward 421 and 394; but 4 x 1024: 41
// and 43, 162 and 165)
bool split_tiles(int64_t blocks, int64_t tiles = 0) { return blocks <= 256 || (blocks <= 512 && tiles >= 16); }

// q, kv, k_rope of latent attention: (nope, value) head dims, refused where no kernel is built for them
std::pair<int, int> check_latent(const at::Tensor& q, const at::Tensor& kv, const at::Tensor& k_rope, const char* op) {
  check_rows(q, q, op, "q", 4);
  check_rows(kv, q, op, "kv", 4);
  check_rows(k_rope, q, op, "k_rope", 3);
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2);
  TORCH_CHECK(kv.size(0) == B && kv.size(1) == S && kv.size(2) == H, op, ": kv must be [B, S, H, nope + value]");
  TORCH_CHECK(k_rope.size(0) == B && k_rope.size(1) == S, op, ": k_rope must be [B, S, rope]");
  const int64_t dr = k_rope.size(2), dn = q.size(3) - dr, dv = kv.size(3) - dn;
  TORCH_CHECK((dn == 128 && dr == 64 && dv == 128) || (dn == 64 && dr == 32 && dv == 64), op,
              ": head dims (nope, rope, value) must be (128, 64, 128) or (64, 32, 64), got (", dn, ", ", dr, ", ", dv, ")");
  TORCH_CHECK(S < INT32_MAX / 4 && B * H < INT32_MAX, op, ": too many rows");
  return {(int)dn, (int)dv};
}

template <typename E>
SharedArgs<E> latent_args(const at::Tensor& q, const at::Tensor& kv, const at::Tensor& kr, int dn, const int* lens,
                          double scale, bool causal) {
  SharedArgs<E> p{};
  p.q = ptr<E>(q), p.k = ptr<E>(kv), p.v = ptr<E>(kv) + dn, p.kr = ptr<E>(kr);
  p.q_sb = stride_of(q, 0), p.q_ss = stride_of(q, 1), p.q_sh = stride_of(q, 2);
  p.k_sb = p.v_sb = stride_of(kv, 0), p.k_ss = p.v_ss = stride_of(kv, 1), p.k_sh = p.v_sh = stride_of(kv, 2);
  p.kr_sb = stride_of(kr, 0), p.kr_ss = stride_of(kr, 1);
  p.lens = lens;
  p.B = q.size(0), p.S = q.size(1), p.Hq = p.Hkv = q.size(2), p.n = 1;
  p.scale = scale, p.scale_log2 = scale * kLog2e, p.neg_inv_scale = -1.0 / scale;
  p.causal = causal;
  return p;
}

void check_prefix(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& pk,
                  const at::Tensor& pv, const char* op) {
  check_rows(q, q, op, "q", 4);
  check_rows(k, q, op, "k", 4);
  check_rows(v, q, op, "v", 4);
  check_rows(pk, q, op, "prefix_k", 4);
  check_rows(pv, q, op, "prefix_v", 4);
  const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(2), G = pk.size(0);
  TORCH_CHECK(D == 64 || D == 128, op, ": head dim must be 64 or 128, got ", D);
  TORCH_CHECK(k.size(0) == B && k.size(1) == S && k.size(3) == D && v.sizes() == k.sizes(), op,
              ": k and v must be [B, S, Hkv, D]");
  TORCH_CHECK(pk.size(2) == Hkv && pk.size(3) == D && pv.sizes() == pk.sizes(), op,
              ": prefix_k and prefix_v must be [G, P, Hkv, D]");
  TORCH_CHECK(Hkv > 0 && Hq % Hkv == 0, op, ": q heads must be a multiple of the kv heads");
  TORCH_CHECK(G > 0 && B % G == 0, op, ": the batch must hold equally many sequences of each prefix");
  TORCH_CHECK(S < INT32_MAX / 4 && pk.size(1) < INT32_MAX / 2 && B * Hq < INT32_MAX, op, ": too many rows");
}

template <typename E>
SharedArgs<E> prefix_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& pk,
                          const at::Tensor& pv, const int* lens, const int* plens, double scale, bool causal) {
  SharedArgs<E> p{};
  p.q = ptr<E>(q), p.k = ptr<E>(k), p.v = ptr<E>(v), p.pk = ptr<E>(pk), p.pv = ptr<E>(pv);
  p.q_sb = stride_of(q, 0), p.q_ss = stride_of(q, 1), p.q_sh = stride_of(q, 2);
  p.k_sb = stride_of(k, 0), p.k_ss = stride_of(k, 1), p.k_sh = stride_of(k, 2);
  p.v_sb = stride_of(v, 0), p.v_ss = stride_of(v, 1), p.v_sh = stride_of(v, 2);
  p.pk_sb = stride_of(pk, 0), p.pk_ss = stride_of(pk, 1), p.pk_sh = stride_of(pk, 2);
  p.pv_sb = stride_of(pv, 0), p.pv_ss = stride_of(pv, 1), p.pv_sh = stride_of(pv, 2);
  p.lens = lens, p.plens = plens;
  p.B = q.size(0), p.S = q.size(1), p.Hq = q.size(2), p.Hkv = k.size(2), p.P = pk.size(1), p.n = p.B / pk.size(0);
  p.scale = scale, p.scale_log2 = scale * kLog2e, p.neg_inv_scale = -1.0 / scale;
  p.causal = causal;
  return p;
}

}  // namespace

// q [B, S, H, nope + rope], kv [B, S, H, nope + value], k_rope [B, S, rope] -> out [B, S, H, value], lse [B, H, S]
std::tuple<at::Tensor, at::Tensor> dlgm_latent_attn_fwd(const at::Tensor& q, const at::Tensor& kv,
                                                        const at::Tensor& k_rope, double softmax_scale, bool causal,
                                                        const c10::optional<at::Tensor>& lens) {
  const char* op = "latent_attn_fwd";
  const auto [dn, dv] = check_latent(q, kv, k_rope, op);
  check_scale(softmax_scale, op);
  const int* lp = check_lens(lens, q, q.size(0), op, "lens");
  const c10::DeviceGuard guard(q.device());
  auto out = at::empty({q.size(0), q.size(1), q.size(2), dv}, q.options());
  auto lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  if (out.numel() == 0) return {out, lse};
  const int64_t blocks = check_blocks(q.size(0) * q.size(2) * ((q.size(1) + kBQ - 1) / kBQ), op);
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    auto p = latent_args<E>(q, kv, k_rope, dn, lp, softmax_scale, causal);
    p.out = ptr<E>(out), p.lse = lse.data_ptr<float>();
    auto run = [&](auto sc) {
      constexpr int SP = decltype(sc)::value;
      if (dn == 128) shared_fwd_kernel<E, 128, 64, 128, false, SP><<<blocks, kThreads * SP, 0, stream>>>(p);
      else shared_fwd_kernel<E, 64, 32, 64, false, SP><<<blocks, kThreads * SP, 0, stream>>>(p);
    };
    if (split_tiles(blocks, (p.S + kBQ - 1) / kBQ)) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 1>{});
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return {out, lse};
}

// Gradients of q, kv and k_rope (contiguous, in their shapes).
std::tuple<at::Tensor, at::Tensor, at::Tensor> dlgm_latent_attn_bwd(const at::Tensor& dout, const at::Tensor& q,
                                                                    const at::Tensor& kv, const at::Tensor& k_rope,
                                                                    const at::Tensor& out, const at::Tensor& lse,
                                                                    double softmax_scale, bool causal,
                                                                    const c10::optional<at::Tensor>& lens) {
  const char* op = "latent_attn_bwd";
  const auto [dn, dv] = check_latent(q, kv, k_rope, op);
  check_scale(softmax_scale, op);
  check_rows(dout, q, op, "dout", 4);
  check_rows(out, q, op, "out", 4);
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2), dr = k_rope.size(2);
  TORCH_CHECK(out.is_contiguous() && out.sizes() == at::IntArrayRef({B, S, H, dv}) && dout.sizes() == out.sizes(), op,
              ": out must be the contiguous [B, S, H, value] of the forward, dout of its shape");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.sizes() == at::IntArrayRef({B, H, S}),
              op, ": lse must be the forward's [B, H, S]");
  const int* lp = check_lens(lens, q, B, op, "lens");
  const c10::DeviceGuard guard(q.device());
  auto dq = at::empty({B, S, H, dn + dr}, q.options());
  auto dkv = at::empty({B, S, H, dn + dv}, q.options());
  auto dkr = at::empty({B, S, dr}, q.options());
  if (B == 0 || S == 0) return {dq, dkv, dkr};
  if (H == 0) return {dq, dkv, dkr.zero_()};
  const auto f32 = q.options().dtype(at::kFloat);
  auto rows = at::empty({2, B, H, S}, f32);
  auto dkr_part = at::empty({H, B, S, dr}, f32);
  const int64_t blocks = check_blocks(2 * B * H * ((S + kBQ - 1) / kBQ), op) / 2;  // dK/dV: of 512 threads
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    auto p = latent_args<E>(q, kv, k_rope, dn, lp, softmax_scale, causal);
    p.o = ptr<E>(out), p.dout = ptr<E>(dout), p.lse = lse.data_ptr<float>(), p.rows = rows.data_ptr<float>();
    p.do_sb = stride_of(dout, 0), p.do_ss = stride_of(dout, 1), p.do_sh = stride_of(dout, 2);
    p.dq = ptr<E>(dq), p.dk = ptr<E>(dkv), p.dv = ptr<E>(dkv) + dn;
    p.dk_ss = p.dv_ss = H * (dn + dv), p.dk_sh = p.dv_sh = dn + dv;
    p.dkr_part = dkr_part.data_ptr<float>();
    auto dq_pass = [&](auto sc) {
      constexpr int SP = decltype(sc)::value;
      if (dn == 128) shared_bwd_dq_kernel<E, 128, 64, 128, false, SP><<<blocks, kThreads * SP, 0, stream>>>(p);
      else shared_bwd_dq_kernel<E, 64, 32, 64, false, SP><<<blocks, kThreads * SP, 0, stream>>>(p);
    };
    if (split_tiles(blocks, (p.S + kBQ - 1) / kBQ)) dq_pass(std::integral_constant<int, 2>{});
    else dq_pass(std::integral_constant<int, 1>{});
    if (dn == 128) {
      latent_bwd_dkdv_kernel<E, 128, 64, 128><<<blocks, kKvThreads, 0, stream>>>(p);
    } else {
      latent_bwd_dkdv_kernel<E, 64, 32, 64><<<blocks, kKvThreads, 0, stream>>>(p);
    }
    SumArgs<E> a{};
    a.part[0] = p.dkr_part, a.out[0] = ptr<E>(dkr), a.n[0] = B * S * dr, a.parts[0] = H;
    const int64_t grid = std::min<int64_t>((a.n[0] / 8 + 255) / 256, 4096);
    sum_parts_kernel<E><<<grid, 256, 0, stream>>>(a);
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return {dq, dkv, dkr};
}

// q [B, S, Hq, D], k/v [B, S, Hkv, D], prefix_k/v [G, P, Hkv, D], B = G n -> out [B, S, Hq, D], lse [B, Hq, S]
std::tuple<at::Tensor, at::Tensor> dlgm_prefix_attn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                        const at::Tensor& prefix_k, const at::Tensor& prefix_v,
                                                        double softmax_scale, bool causal,
                                                        const c10::optional<at::Tensor>& lens,
                                                        const c10::optional<at::Tensor>& prefix_lens) {
  const char* op = "prefix_attn_fwd";
  check_prefix(q, k, v, prefix_k, prefix_v, op);
  check_scale(softmax_scale, op);
  const int* lp = check_lens(lens, q, q.size(0), op, "lens");
  const int* pp = check_lens(prefix_lens, q, prefix_k.size(0), op, "prefix_lens");
  const c10::DeviceGuard guard(q.device());
  auto out = at::empty(q.sizes(), q.options());
  auto lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  if (out.numel() == 0) return {out, lse};
  const int64_t blocks = check_blocks(q.size(0) * q.size(2) * ((q.size(1) + kBQ - 1) / kBQ), op);
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    auto p = prefix_args<E>(q, k, v, prefix_k, prefix_v, lp, pp, softmax_scale, causal);
    p.out = ptr<E>(out), p.lse = lse.data_ptr<float>();
    auto run = [&](auto sc) {
      constexpr int SP = decltype(sc)::value;
      if (q.size(3) == 128) shared_fwd_kernel<E, 128, 0, 128, true, SP><<<blocks, kThreads * SP, 0, stream>>>(p);
      else shared_fwd_kernel<E, 64, 0, 64, true, SP><<<blocks, kThreads * SP, 0, stream>>>(p);
    };
    if (split_tiles(blocks)) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 1>{});
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return {out, lse};
}

// Gradients of q, k, v, prefix_k and prefix_v (contiguous, in their shapes).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> dlgm_prefix_attn_bwd(
    const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& prefix_k,
    const at::Tensor& prefix_v, const at::Tensor& out, const at::Tensor& lse, double softmax_scale, bool causal,
    const c10::optional<at::Tensor>& lens, const c10::optional<at::Tensor>& prefix_lens) {
  const char* op = "prefix_attn_bwd";
  check_prefix(q, k, v, prefix_k, prefix_v, op);
  check_scale(softmax_scale, op);
  check_rows(dout, q, op, "dout", 4);
  check_rows(out, q, op, "out", 4);
  const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(2);
  const int64_t G = prefix_k.size(0), P = prefix_k.size(1), n = B / G;
  TORCH_CHECK(out.is_contiguous() && out.sizes() == q.sizes() && dout.sizes() == q.sizes(), op,
              ": out must be the contiguous [B, S, Hq, D] of the forward, dout of its shape");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.sizes() == at::IntArrayRef({B, Hq, S}),
              op, ": lse must be the forward's [B, Hq, S]");
  const int* lp = check_lens(lens, q, B, op, "lens");
  const int* pp = check_lens(prefix_lens, q, G, op, "prefix_lens");
  const c10::DeviceGuard guard(q.device());
  auto dq = at::empty(q.sizes(), q.options());
  auto dk = at::empty(k.sizes(), q.options()), dv = at::empty(k.sizes(), q.options());
  auto dpk = at::empty(prefix_k.sizes(), q.options()), dpv = at::empty(prefix_k.sizes(), q.options());
  if (B == 0 || S == 0 || Hq == 0) return {dq.zero_(), dk.zero_(), dv.zero_(), dpk.zero_(), dpv.zero_()};
  const auto f32 = q.options().dtype(at::kFloat);
  auto rows = at::empty({2, B, Hq, S}, f32);
  const int64_t group = Hq / Hkv, hp = group % 2 == 0 ? 2 : 1, gp = group / hp;
  const int64_t pkt = (P + kBQ - 1) / kBQ;
  // a group's sequences are cut into parts until the prefix's workgroups fill the chip twice over (256 CUs, two each);
  // a part costs an fp32 copy of the prefix's gradient, so no more parts than that (16 x 256 queries over 1024 + 256 keys,
  // 16/4 heads, the whole backward: 450 us uncut, 214 so). Two q heads share a workgroup where the group is even: it takes
  // the same time as one each (2050 us at 8 x 1024 over 4096) and half the partial sums' memory.
  const int64_t whole = std::max<int64_t>(1, G * (Hq / hp) * pkt);
  const int64_t nsplit = std::max<int64_t>(1, std::min<int64_t>(n, 1024 / whole));
  at::Tensor dk_part, dv_part, dpk_part, dpv_part;
  if (gp > 1) {
    dk_part = at::empty({gp, B, S, Hkv, D}, f32);
    dv_part = at::empty({gp, B, S, Hkv, D}, f32);
  }
  if (gp * nsplit > 1) {
    dpk_part = at::empty({gp * nsplit, G, P, Hkv, D}, f32);
    dpv_part = at::empty({gp * nsplit, G, P, Hkv, D}, f32);
  }
  const int64_t q_blocks = check_blocks(B * Hq * ((S + kBQ - 1) / kBQ), op);
  const int64_t p_blocks = G * (Hq / hp) * nsplit * pkt;
  const int64_t k_blocks = check_blocks(p_blocks + B * (Hq / hp) * ((S + kBQ - 1) / kBQ), op);
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    auto p = prefix_args<E>(q, k, v, prefix_k, prefix_v, lp, pp, softmax_scale, causal);
    p.o = ptr<E>(out), p.dout = ptr<E>(dout), p.lse = lse.data_ptr<float>(), p.rows = rows.data_ptr<float>();
    p.do_sb = stride_of(dout, 0), p.do_ss = stride_of(dout, 1), p.do_sh = stride_of(dout, 2);
    p.dq = ptr<E>(dq), p.dk = ptr<E>(dk), p.dv = ptr<E>(dv), p.dpk = ptr<E>(dpk), p.dpv = ptr<E>(dpv);
    p.nsplit = nsplit, p.prefix_blocks = p_blocks;
    SumArgs<E> a{};
    int sums = 0;
    auto sum = [&](const at::Tensor& part, const at::Tensor& to, int64_t parts) {
      if (!part.defined() || to.numel() == 0) return;
      a.part[sums] = part.data_ptr<float>(), a.out[sums] = ptr<E>(to), a.n[sums] = to.numel(), a.parts[sums] = parts;
      ++sums;
    };
    sum(dk_part, dk, gp), sum(dv_part, dv, gp), sum(dpk_part, dpk, gp * nsplit), sum(dpv_part, dpv, gp * nsplit);
    if (gp > 1) p.dk_part = dk_part.data_ptr<float>(), p.dv_part = dv_part.data_ptr<float>();
    if (gp * nsplit > 1) p.dpk_part = dpk_part.data_ptr<float>(), p.dpv_part = dpv_part.data_ptr<float>();
    auto run = [&](auto dc) {
      constexpr int DD = decltype(dc)::value;
      if (split_tiles(q_blocks)) shared_bwd_dq_kernel<E, DD, 0, DD, true, 2><<<q_blocks, 2 * kThreads, 0, stream>>>(p);
      else shared_bwd_dq_kernel<E, DD, 0, DD, true, 1><<<q_blocks, kThreads, 0, stream>>>(p);
      if (hp == 2) prefix_bwd_dkdv_kernel<E, DD, 2><<<k_blocks, kThreads, 0, stream>>>(p);
      else prefix_bwd_dkdv_kernel<E, DD, 1><<<k_blocks, kThreads, 0, stream>>>(p);
    };
    if (D == 128) run(std::integral_constant<int, 128>{});
    else run(std::integral_constant<int, 64>{});
    if (sums) {
      int64_t most = 0;
      for (int i = 0; i < sums; ++i) most = std::max(most, a.n[i]);
      const dim3 grid(std::min<int64_t>((most / 8 + 255) / 256, 4096), sums);
      sum_parts_kernel<E><<<grid, 256, 0, stream>>>(a);
    }
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return {dq, dk, dv, dpk, dpv};
}
