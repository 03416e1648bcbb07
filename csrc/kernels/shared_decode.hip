// Attention whose keys and values are shared, single-token forms over a cache (gfx950).
//
//  * latent attention, absorbed: with W_k[h] (nope x r) and W_v[h] (value x r) the up-projections of head h,
//      s[h,t] = scale (q_nope[h] W_k[h] . c[t] + q_rope[h] . k_rope[t]),   o[h] = W_v[h] sum_t softmax(s)[h,t] c[t]
//    so the cache holds ONE row [c | k_rope] a token and all heads read it. Three launches: absorb (q_nope W_k), attend
//    (the cache, split over its length), project (join the parts, W_v).
//  * a batch over a shared prefix: the n sequences of a group and the q heads of a kv head are the rows of one product
//    with the prefix, which is read once for all of them; each sequence then reads its own cache. Two launches: attend
//    (prefix parts and own parts side by side), join.
//
// Both are bound by reading the cache once (a row of it meets 2 H (2r + dr) operations in the latent form, 4 rows D in the
// other), so the work is cut along the length until the chip is full, each sequence by its own length; a part keeps its
// running maximum, sum and unnormalised output in fp32, and the parts are joined in a fixed order (no atomics).
#include <torch/all.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <type_traits>
#include "dlgm_attn.h"
#include "dlgm_attn_host.h"

using namespace dlgm;

namespace {

// f32x8 of 8 consecutive floats, 16-byte aligned
__device__ __forceinline__ f32x8 load8(const float* p) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
  return (f32x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// ---- latent attention -------------------------------------------------------------------------

template <typename E>
struct LatentArgs {
  const E *q, *cache, *w;
  E *qa, *out;      // qa [B, H, r]: q_nope W_k; out [B, H, value]
  float *o, *ml;    // parts [B, H, ns, r] and [B, H, ns, 2] (running maximum in the log2 domain, sum)
  const int* lens;  // [B]
  int64_t q_sb, q_sh, c_sb, c_ss, w_ss;
  int B, H, L, dn, dv, ns;
  float scale_log2;

  __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), L); }
};

// qa[b, h, :] = q_nope[b, h, :] W_k[h]: one workgroup per (head, 128 latent columns), a wave per 32 of them, 32 sequences
// a step. qa is rounded to the 16-bit type: it is the matrix operand of the scores, as q is in the expanded form.
template <typename E, int DN>
__global__ __launch_bounds__(kThreads) void latent_absorb_kernel(LatentArgs<E> p, int R) {
  __shared__ __attribute__((aligned(16))) E img[DN * 128];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int nc = R / 128, head = blockIdx.x / nc, c0 = blockIdx.x % nc * 128;
  const RowTile<E, 128, DN, 2> wt(w, lane);
  wt.issue(img, p.w + (int64_t)head * (p.dn + p.dv) * p.w_ss + c0, p.w_ss, DN, w);
  vm_drain();
  __syncthreads();
  const TrFrag<128, 2> wf(h, i16, g4);
  vec8_t<E> a[DN / 16];
#pragma unroll
  for (int s = 0; s < DN / 16; ++s) a[s] = wf.read(img, w, 16 * s);
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int b = b0 + r;
    const E* q = p.q + b * p.q_sb + head * p.q_sh;
    f32x16 acc = (f32x16)(0.f);
#pragma unroll
    for (int s = 0; s < DN / 16; ++s) {
      vec8_t<E> f = (vec8_t<E>)((E)0.f);
      if (b < p.B)  // the k order of the transposed read: rows 16 s + 4 h .. +3, then the same + 8
        f = cat(*reinterpret_cast<const vec4_t<E>*>(q + 16 * s + 4 * h), *reinterpret_cast<const vec4_t<E>*>(q + 16 * s + 8 + 4 * h));
      acc = mfma32(a[s], f, acc);
    }
    const f32x16 acc1[1] = {acc};
    store_rows_bf16<1>(p.qa + ((int64_t)b * p.H + head) * R + c0 + 32 * w, acc1, 1.f, h, b < p.B);
  }
}

// One workgroup per (sequence, 64 heads, part of its length): tiles of 64 cache rows by LDS-DMA, one ahead. Scores: wave
// (u, hb) takes 32 rows x 32 heads over all r + dr columns, its q operand in registers. Outputs: each wave takes r / 4
// latent columns of all 64 heads; the weights pass through LDS in fragment order. 64 heads a workgroup keep the cache rows'
// LDS reads (36 KiB a wave and tile at r 512) below the matrix time (68 MFMA) with one wave a SIMD.
template <typename E, int R, int DR>
__global__ __launch_bounds__(kThreads, 1) void latent_attend_kernel(LatentArgs<E> p) {
  constexpr int NI = R / 128, KR = R / 16, KK = KR + DR / 16;  // images, k-steps
  constexpr int TI = 64 * 128, SLOT = 64 * (R + DR);
  constexpr int DT = R / 128;  // 32-column output tiles of a wave
  __shared__ __attribute__((aligned(16))) E smem[2 * SLOT];
  __shared__ __attribute__((aligned(16))) E pbuf[8 * 512];  // [u][s2][hb] fragments of 64 lanes x 8
  __shared__ float smax[2][64], ssum[2][64];

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int u = w & 1, hb = w >> 1;
  const int nhb = (p.H + 63) / 64;
  // head blocks of one (sequence, part) read the same rows: they follow each other on one XCD
  const int work = xcd_remap(blockIdx.x, gridDim.x);
  const int head0 = work % nhb * 64, part = work / nhb % p.ns, b = work / nhb / p.ns;
  const int len = p.len(b);
  const int tiles = (len + 63) / 64;
  const int t0 = (int)((int64_t)tiles * part / p.ns), t1 = (int)((int64_t)tiles * (part + 1) / p.ns);

  const int head = head0 + 32 * hb + r;
  vec8_t<E> qf[KK];
  {
    const E* qa = p.qa + ((int64_t)b * p.H + head) * R + 8 * h;
    const E* qr = p.q + b * p.q_sb + head * p.q_sh + p.dn + 8 * h;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[kk] = row8(kk < KR ? qa + 16 * kk : qr + 16 * (kk - KR), head < p.H);
  }
  const RowTile<E, 128, 64, 1> ct(w, lane);
  const RowTile<E, DR, 64, 0> rt(w, lane);
  const E* cb = p.cache + b * p.c_sb;
  auto stage = [&](int buf, int t) {
    E* img = smem + buf * SLOT;
    const E* base = cb + (int64_t)t * 64 * p.c_ss;
#pragma unroll
    for (int i = 0; i < NI; ++i) ct.issue(img + i * TI, base + 128 * i, p.c_ss, len - t * 64, w);
    rt.issue(img + NI * TI, base + R, p.c_ss, len - t * 64, w);
  };

  f32x16 o[2][DT];  // [head block][column tile]
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = (f32x16)(0.f);
  RowFrag<128, 1> cf(r, h);
  RowFrag<DR, 0> rf(r, h);
  TrFrag<128, 1> vf(h, i16, g4);
  float m_run[2] = {-INFINITY, -INFINITY}, l_run = 0.f;  // maxima of heads r and 32 + r; the sum of this wave's rows

  auto tile = [&](auto bufc, int t) {
    constexpr int buf = decltype(bufc)::value;
    vm_drain();
    __syncthreads();
    if (t + 1 < t1) stage(buf ^ 1, t + 1);
    const E* img = smem + buf * SLOT;
    pin(cf.at), pin(rf.at), pin(vf.at);
    f32x16 s = (f32x16)(0.f);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const E* a = kk < KR ? img + kk / 8 * TI + 32 * u * 128 + cf(kk % 8) : img + NI * TI + 32 * u * DR + rf(kk - KR);
      s = mfma32(lds_read_b128(a), qf[kk], s);
    }
    if (uniform(t * 64 + 64 > len)) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (t * 64 + 32 * u + (i & 3) + 8 * (i >> 2) + 4 * h >= len) s[i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, swap_halves(mx)) * p.scale_log2;
    if (h == 0) smax[u][32 * hb + r] = mx;
    __syncthreads();
    // every wave follows the maxima of all 64 heads, so the weights of a tile share one reference
    float mt[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) mt[x] = fmaxf(smax[0][32 * x + r], smax[1][32 * x + r]);
    if (__any(mt[0] > m_run[0] + kRescaleLog2 || mt[1] > m_run[1] + kRescaleLog2)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float m_new = fmaxf(m_run[x], mt[x]);
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run[x] - m_new);
        m_run[x] = m_new;
        if (x == hb) l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= alpha;
      }
    }
    const float m_own = hb ? m_run[1] : m_run[0];
    const float m_use = m_own == -INFINITY ? 0.f : m_own;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = fast_exp2(s[i] * p.scale_log2 - m_use);
      l_run += s[i];
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
      *reinterpret_cast<vec8_t<E>*>(pbuf + ((2 * u + s2) * 2 + hb) * 512 + lane * 8) = pack8<E>(s, 8 * s2);
    __syncthreads();
    vec8_t<E> pf[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int k = 0; k < 4; ++k) pf[x][k] = lds_read_b128(pbuf + (2 * k + x) * 512 + lane * 8);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int col = w * DT + dt;  // 32-column tile of the latent vector
      const E* vi = img + col / 4 * TI;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const vec8_t<E> a = vf.read(vi, col % 4, 16 * k);
        o[0][dt] = mfma32(a, pf[0][k], o[0][dt]);
        o[1][dt] = mfma32(a, pf[1][k], o[1][dt]);
      }
    }
  };
  if (t0 < t1) stage(0, t0);
  for (int t = t0; t < t1; t += 2) {
    tile(std::integral_constant<int, 0>{}, t);
    if (t + 1 < t1) tile(std::integral_constant<int, 1>{}, t + 1);
  }

  const float l_half = l_run + swap_halves(l_run);
  if (h == 0) ssum[u][32 * hb + r] = l_half;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int hd = head0 + 32 * x + r;
    if (hd >= p.H) continue;
    const int64_t slot = ((int64_t)b * p.H + hd) * p.ns + part;
    if (w == 0 && h == 0) {
      p.ml[2 * slot] = m_run[x];
      p.ml[2 * slot + 1] = ssum[0][32 * x + r] + ssum[1][32 * x + r];
    }
    if (t0 < t1) store_rows_f32<DT>(p.o + slot * R + w * DT * 32, o[x], 1.f, h);  // an empty part is not read
  }
}

// One workgroup per (head, 32 sequences): join the parts into the latent output (16 bits in LDS, the operand of the
// product), then out = W_v[h] o.
template <typename E, int R, int DV>
__global__ __launch_bounds__(kThreads) void latent_project_kernel(LatentArgs<E> p) {
  constexpr int LD = R + 8;
  __shared__ __attribute__((aligned(16))) E ol[32 * LD];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int head = blockIdx.x % p.H, b0 = blockIdx.x / p.H * 32;
  const int col = lane * 8;
  for (int k = w; k < 32; k += 4) {
    const int b = b0 + k;
    f32x8 acc = (f32x8)(0.f);
    float l = 0.f;
    if (b < p.B) {
      const int64_t slot = ((int64_t)b * p.H + head) * p.ns;
      float m = -INFINITY;
      for (int s = 0; s < p.ns; ++s) m = fmaxf(m, p.ml[2 * (slot + s)]);
      for (int s = 0; s < p.ns; ++s) {
        const float ls = p.ml[2 * (slot + s) + 1];
        if (ls == 0.f) continue;  // an empty part (a NaN sum is none)
        const float f = fast_exp2(p.ml[2 * (slot + s)] - m);
        l += f * ls;
        if (col < R) acc += load8(p.o + (slot + s) * R + col) * f;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a sequence without keys: zeros
    if (col < R) store8f(ol + k * LD + col, acc * inv);
  }
  __syncthreads();
  if (w >= DV / 32) return;
  const E* wv = p.w + ((int64_t)head * (p.dn + p.dv) + p.dn + 32 * w + r) * p.w_ss + 8 * h;
  f32x16 acc = (f32x16)(0.f);
#pragma unroll 8
  for (int kk = 0; kk < R / 16; ++kk)
    acc = mfma32(*reinterpret_cast<const vec8_t<E>*>(wv + 16 * kk), lds_read_b128(ol + r * LD + 16 * kk + 8 * h), acc);
  const f32x16 acc1[1] = {acc};
  store_rows_bf16<1>(p.out + ((int64_t)(b0 + r) * p.H + head) * DV + 32 * w, acc1, 1.f, h, b0 + r < p.B);
}

// ---- shared prefix ------------------------------------------------------------------------------

template <typename E>
struct PrefixArgs {
  const E *q, *k, *v, *pk, *pv;
  E* out;                   // [B, Hq, D]
  float *o, *ml;            // parts [B, Hq, np + no, D] and [B, Hq, np + no, 2]
  const int *lens, *plens;  // [B], [G] (null: all)
  int64_t q_sb, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  int64_t pk_sb, pk_ss, pk_sh, pv_sb, pv_ss, pv_sh;
  int B, Hq, Hkv, L, P, G, n;
  int np, no;          // parts of the prefix and of a sequence's own cache
  int prw, orw;        // waves along the rows (1, 2 or 4) of prefix and own workgroups; the others share the keys
  int prb, orb;        // row blocks of 32 prw / 32 orw rows
  int prefix_blocks;
  float scale_log2;
};

// One workgroup per (kv head, block of rows, part of a key range): 128 keys a step by LDS-DMA, one step ahead. The rows
// are (sequence of the group, q head of the kv head) for the prefix and the q heads for a sequence's own keys. rw of the 4
// waves stand along the rows, so few rows leave the waves to share the 128 keys (joined through LDS at the end) and many
// rows read each key once for 128 of them.
template <typename E, int D>
__global__ __launch_bounds__(kThreads, 1) void prefix_attend_kernel(PrefixArgs<E> p) {
  constexpr int KK = D / 16, DT = D / 32, KEYS = 128;
  constexpr int TI = KEYS * D, SLOT = 2 * TI;
  constexpr int LDO = D + 4;
  __shared__ __attribute__((aligned(16))) E smem[2 * SLOT];
  __shared__ float sm[4][32], sl[4][32];
  static_assert(sizeof(E) * 2 * SLOT >= 4 * 32 * LDO * 4, "the joined rows fit the tiles' space");

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int rep = p.Hq / p.Hkv;
  const bool pre = (int)blockIdx.x < p.prefix_blocks;
  int rw, rb, part, nparts, hk, b0, nrows, len;  // first sequence, rows in all, keys
  const E *kb, *vb;
  int64_t k_ss, v_ss;
  if (pre) {
    // row blocks of one part read the same keys: they follow each other on one XCD
    int x = xcd_remap(blockIdx.x, p.prefix_blocks);
    rw = p.prw, nparts = p.np;
    rb = x % p.prb, x /= p.prb;
    part = x % p.np, x /= p.np;
    hk = x % p.Hkv;
    const int g = x / p.Hkv;
    b0 = g * p.n, nrows = p.n * rep;
    len = p.plens ? min(max(p.plens[g], 0), p.P) : p.P;
    kb = p.pk + g * p.pk_sb + hk * p.pk_sh, vb = p.pv + g * p.pv_sb + hk * p.pv_sh;
    k_ss = p.pk_ss, v_ss = p.pv_ss;
  } else {
    int x = xcd_remap(blockIdx.x - p.prefix_blocks, gridDim.x - p.prefix_blocks);
    rw = p.orw, nparts = p.no;
    rb = x % p.orb, x /= p.orb;
    part = x % p.no, x /= p.no;
    hk = x % p.Hkv;
    b0 = x / p.Hkv, nrows = rep;
    len = min(max(p.lens[b0], 0), p.L);
    kb = p.k + b0 * p.k_sb + hk * p.k_sh, vb = p.v + b0 * p.v_sb + hk * p.v_sh;
    k_ss = p.k_ss, v_ss = p.v_ss;
  }
  const int kw = w / rw;  // this wave's share of a step's keys: rw blocks of 32 from block kw rw on
  const int idx = (rb * rw + w % rw) * 32 + r, seq = b0 + idx / rep, hq = hk * rep + idx % rep;
  const bool ok = idx < nrows;
  const int steps = (len + KEYS - 1) / KEYS;
  const int t0 = (int)((int64_t)steps * part / nparts), t1 = (int)((int64_t)steps * (part + 1) / nparts);

  vec8_t<E> qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qf[kk] = row8(p.q + seq * p.q_sb + hq * p.q_sh + 16 * kk + 8 * h, ok);
  const RowTile<E, D, KEYS, 0> kt(w, lane);
  const RowTile<E, D, KEYS, 2> vt(w, lane);
  auto stage = [&](int buf, int t) {
    E* img = smem + buf * SLOT;
    kt.issue(img, kb + (int64_t)t * KEYS * k_ss, k_ss, len - t * KEYS, w);
    vt.issue(img + TI, vb + (int64_t)t * KEYS * v_ss, v_ss, len - t * KEYS, w);
  };
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = (f32x16)(0.f);
  float m_run = -INFINITY, l_run = 0.f;
  const RowFrag<D, 0> kf(r, h);
  const TrFrag<D, 2> vf(h, i16, g4);
  if (t0 < t1) stage(0, t0);
  for (int t = t0; t < t1; ++t) {
    vm_drain();
    __syncthreads();
    const int buf = (t - t0) & 1;
    if (t + 1 < t1) stage(buf ^ 1, t + 1);
    for (int x = 0; x < rw; ++x) {
      const int blk = kw * rw + x, key0 = t * KEYS + 32 * blk;
      if (key0 >= len) break;
      const E* ki = smem + buf * SLOT + blk * 32 * D;
      const E* vi = ki + TI;
      f32x16 s = (f32x16)(0.f);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) s = mfma32(lds_read_b128(ki + kf(kk)), qf[kk], s);
      if (uniform(key0 + 32 > len)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + (i & 3) + 8 * (i >> 2) + 4 * h >= len) s[i] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
      mx = fmaxf(mx, swap_halves(mx)) * p.scale_log2;
      if (__any(mx > m_run + kRescaleLog2)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      }
      const float m_use = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = fast_exp2(s[i] * p.scale_log2 - m_use);
        l_run += s[i];
      }
      const vec8_t<E> pf[2] = {pack8<E>(s, 0), pack8<E>(s, 8)};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) o[dt] = mfma32(vf.read(vi, dt, 16 * s2), pf[s2], o[dt]);
    }
  }

  const int slots = p.np + p.no, slot = pre ? part : p.np + part;
  const int64_t at = ((int64_t)seq * p.Hq + hq) * slots + slot;
  float l = l_run + swap_halves(l_run);
  if (rw == 4) {  // no other wave has these rows
    if (ok) {
      if (h == 0) p.ml[2 * at] = m_run, p.ml[2 * at + 1] = l;
      if (t0 < t1) store_rows_f32<DT>(p.o + at * D, o, 1.f, h);  // an empty part is not read
    }
    return;
  }
  if (h == 0) sm[w][r] = m_run, sl[w][r] = l;
  __syncthreads();  // also: the last tiles have been read
  float m = -INFINITY;
  for (int x = w % rw; x < 4; x += rw) m = fmaxf(m, sm[x][r]);
  const float f = l == 0.f ? 0.f : fast_exp2(m_run - m);
  float* joined = reinterpret_cast<float*>(smem);
  store_rows_f32<DT>(joined + (w * 32 + r) * LDO, o, f, h);
  __syncthreads();
  // the rw blocks of 32 rows, summed over the 4 / rw waves that shared their keys
  for (int i = threadIdx.x; i < rw * 32 * (D / 4); i += kThreads) {
    const int row = i / (D / 4), c = i % (D / 4) * 4, x0 = row >> 5, rr = row & 31;
    const int id = (rb * rw + x0) * 32 + rr;
    if (id >= nrows) break;
    float mm = -INFINITY, ll = 0.f;
    f32x4 acc = (f32x4)(0.f);
    for (int x = x0; x < 4; x += rw) mm = fmaxf(mm, sm[x][rr]);
    for (int x = x0; x < 4; x += rw) {
      ll += sl[x][rr] == 0.f ? 0.f : sl[x][rr] * fast_exp2(sm[x][rr] - mm);
      acc += *reinterpret_cast<const f32x4*>(joined + (x * 32 + rr) * LDO + c);
    }
    const int64_t a = ((int64_t)(b0 + id / rep) * p.Hq + hk * rep + id % rep) * slots + slot;
    if (c == 0) p.ml[2 * a] = mm, p.ml[2 * a + 1] = ll;
    if (t0 < t1) *reinterpret_cast<f32x4*>(p.o + a * D + c) = acc;
  }
}

// One workgroup per (sequence, q head): its waves take the parts in turn, then the four sums are added.
template <typename E, int D>
__global__ __launch_bounds__(kThreads) void prefix_join_kernel(PrefixArgs<E> p) {
  constexpr int V = D / 64;  // columns of a lane
  __shared__ float red[4][D], sl[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int slots = p.np + p.no;
  const int64_t row = blockIdx.x, base = row * slots;
  float m = -INFINITY, l = 0.f, acc[V] = {};
  for (int s = 0; s < slots; ++s) m = fmaxf(m, p.ml[2 * (base + s)]);
  for (int s = w; s < slots; s += 4) {
    const float ls = p.ml[2 * (base + s) + 1];
    if (ls == 0.f) continue;  // an empty part (a NaN sum is none)
    const float f = fast_exp2(p.ml[2 * (base + s)] - m);
    l += f * ls;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] += f * p.o[(base + s) * D + lane * V + j];
  }
#pragma unroll
  for (int j = 0; j < V; ++j) red[w][lane * V + j] = acc[j];
  if (lane == 0) sl[w] = l;
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int c = threadIdx.x;
  const float lt = sl[0] + sl[1] + sl[2] + sl[3];
  const float o = red[0][c] + red[1][c] + red[2][c] + red[3][c];
  p.out[row * D + c] = (E)(lt == 0.f ? 0.f : o / lt);  // a row without keys: zeros
}

// how many parts a length of `steps` steps is cut into so that `items` such lengths give about `want` workgroups
int64_t parts_of(int64_t steps, int64_t items, int64_t want) {
  const int64_t most = 64;  // a join reads every part of a row
  return std::max<int64_t>(1, std::min({steps, most, (want + items - 1) / std::max<int64_t>(1, items)}));
}

// waves along the rows: as many as the rows fill (a step's keys are shared by the rest)
int row_waves(int64_t rows) { return rows > 64 ? 4 : rows > 32 ? 2 : 1; }

}  // namespace

// q [B, H, nope + rope], cache [B, L, r + rope], lens int32 [B], w_kv [H (nope + value), r] -> out [B, H, value]
at::Tensor dlgm_latent_attn_decode(const at::Tensor& q, const at::Tensor& cache, const at::Tensor& lens,
                                   const at::Tensor& w_kv, double softmax_scale) {
  const char* op = "latent_attention_decode";
  check_rows(q, q, op, "q", 3);
  check_rows(cache, q, op, "cache", 3);
  check_rows(w_kv, q, op, "w_kv", 2);
  check_scale(softmax_scale, op);
  const int64_t B = q.size(0), H = q.size(1), L = cache.size(1), r = w_kv.size(1), dr = cache.size(2) - r;
  TORCH_CHECK(cache.size(0) == B, op, ": cache must hold one sequence per row of q");
  TORCH_CHECK(H > 0 && w_kv.size(0) % H == 0, op, ": w_kv must have nope + value rows per head");
  const int64_t dn = q.size(2) - dr, dv = w_kv.size(0) / H - dn;
  TORCH_CHECK((r == 256 || r == 512) && ((dn == 128 && dr == 64 && dv == 128) || (dn == 64 && dr == 32 && dv == 64)), op,
              ": latent size must be 256 or 512 and head dims (nope, rope, value) (128, 64, 128) or (64, 32, 64), got ", r,
              " and (", dn, ", ", dr, ", ", dv, ")");
  TORCH_CHECK(L < INT32_MAX / 2 && B * H < INT32_MAX / 64, op, ": too many rows");
  const int* lp = check_lens(lens, q, B, op, "lens");
  TORCH_CHECK(lp != nullptr || B == 0, op, ": lens is required");
  const c10::DeviceGuard guard(q.device());
  auto out = at::empty({B, H, dv}, q.options());
  if (B == 0) return out;
  if (L == 0) return out.zero_();
  const int64_t nhb = (H + 63) / 64;
  const int64_t ns = parts_of((L + 63) / 64, B * nhb, 256);
  auto qa = at::empty({B, H, r}, q.options());
  auto o = at::empty({B, H, ns, r}, q.options().dtype(at::kFloat));
  auto ml = at::empty({B, H, ns, 2}, q.options().dtype(at::kFloat));
  const int64_t a_blocks = check_blocks(H * (r / 128), op), t_blocks = check_blocks(B * nhb * ns, op);
  const int64_t p_blocks = check_blocks(H * ((B + 31) / 32), op);
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    LatentArgs<E> p{};
    p.q = ptr<E>(q), p.cache = ptr<E>(cache), p.w = ptr<E>(w_kv), p.qa = ptr<E>(qa), p.out = ptr<E>(out);
    p.o = o.data_ptr<float>(), p.ml = ml.data_ptr<float>(), p.lens = lp;
    p.q_sb = q.stride(0), p.q_sh = q.stride(1), p.c_sb = cache.stride(0), p.c_ss = cache.stride(1), p.w_ss = w_kv.stride(0);
    p.B = B, p.H = H, p.L = L, p.dn = dn, p.dv = dv, p.ns = ns;
    p.scale_log2 = softmax_scale * kLog2e;
    auto run = [&](auto rc) {
      constexpr int R = decltype(rc)::value;
      if (dn == 128) {
        latent_absorb_kernel<E, 128><<<a_blocks, kThreads, 0, stream>>>(p, R);
        latent_attend_kernel<E, R, 64><<<t_blocks, kThreads, 0, stream>>>(p);
        latent_project_kernel<E, R, 128><<<p_blocks, kThreads, 0, stream>>>(p);
      } else {
        latent_absorb_kernel<E, 64><<<a_blocks, kThreads, 0, stream>>>(p, R);
        latent_attend_kernel<E, R, 32><<<t_blocks, kThreads, 0, stream>>>(p);
        latent_project_kernel<E, R, 64><<<p_blocks, kThreads, 0, stream>>>(p);
      }
    };
    if (r == 512) run(std::integral_constant<int, 512>{});
    else run(std::integral_constant<int, 256>{});
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return out;
}

// q [B, Hq, D], k/v [B, L, Hkv, D], lens int32 [B], prefix_k/v [G, P, Hkv, D], B = G n -> out [B, Hq, D]
at::Tensor dlgm_prefix_attn_decode(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& lens,
                                   const at::Tensor& prefix_k, const at::Tensor& prefix_v, double softmax_scale,
                                   const c10::optional<at::Tensor>& prefix_lens) {
  const char* op = "prefix_attention_decode";
  check_rows(q, q, op, "q", 3);
  check_rows(k, q, op, "k", 4);
  check_rows(v, q, op, "v", 4);
  check_rows(prefix_k, q, op, "prefix_k", 4);
  check_rows(prefix_v, q, op, "prefix_v", 4);
  check_scale(softmax_scale, op);
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), L = k.size(1), Hkv = k.size(2);
  const int64_t G = prefix_k.size(0), P = prefix_k.size(1);
  TORCH_CHECK(D == 64 || D == 128, op, ": head dim must be 64 or 128, got ", D);
  TORCH_CHECK(k.size(0) == B && k.size(3) == D && v.sizes() == k.sizes(), op, ": k and v must be [B, L, Hkv, D]");
  TORCH_CHECK(prefix_k.size(2) == Hkv && prefix_k.size(3) == D && prefix_v.sizes() == prefix_k.sizes(), op,
              ": prefix_k and prefix_v must be [G, P, Hkv, D]");
  TORCH_CHECK(Hkv > 0 && Hq % Hkv == 0, op, ": q heads must be a multiple of the kv heads");
  TORCH_CHECK(G > 0 && B % G == 0, op, ": the batch must hold equally many sequences of each prefix");
  TORCH_CHECK(L < INT32_MAX / 2 && P < INT32_MAX / 2 && B * Hq < INT32_MAX / 64, op, ": too many rows");
  const int* lp = check_lens(lens, q, B, op, "lens");
  TORCH_CHECK(lp != nullptr || B == 0, op, ": lens is required");
  const int* pp = check_lens(prefix_lens, q, G, op, "prefix_lens");
  const c10::DeviceGuard guard(q.device());
  auto out = at::empty({B, Hq, D}, q.options());
  if (B == 0 || Hq == 0) return out;
  const int64_t rep = Hq / Hkv, n = B / G, psteps = (P + 127) / 128, osteps = (L + 127) / 128;
  const int prw = row_waves(n * rep), orw = row_waves(rep);
  const int64_t prb = (n * rep + 32 * prw - 1) / (32 * prw), orb = (rep + 32 * orw - 1) / (32 * orw);
  // both kinds of workgroup get about the same number of steps, 1024 workgroups in all (256 at a time: the tiles fill a
  // CU's LDS)
  const int64_t pitems = G * Hkv * prb, oitems = B * Hkv * orb;
  const int64_t per = std::max<int64_t>(1, (pitems * psteps + oitems * osteps + 1023) / 1024);
  const int64_t np = P ? parts_of(psteps, 1, (psteps + per - 1) / per) : 0;
  const int64_t no = L ? parts_of(osteps, 1, (osteps + per - 1) / per) : 0;
  if (np + no == 0) return out.zero_();
  auto o = at::empty({B, Hq, np + no, D}, q.options().dtype(at::kFloat));
  auto ml = at::empty({B, Hq, np + no, 2}, q.options().dtype(at::kFloat));
  const int64_t blocks = check_blocks(pitems * np + oitems * no, op);
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    PrefixArgs<E> p{};
    p.q = ptr<E>(q), p.k = ptr<E>(k), p.v = ptr<E>(v), p.pk = ptr<E>(prefix_k), p.pv = ptr<E>(prefix_v), p.out = ptr<E>(out);
    p.o = o.data_ptr<float>(), p.ml = ml.data_ptr<float>(), p.lens = lp, p.plens = pp;
    p.q_sb = q.stride(0), p.q_sh = q.stride(1);
    p.k_sb = k.stride(0), p.k_ss = k.stride(1), p.k_sh = k.stride(2);
    p.v_sb = v.stride(0), p.v_ss = v.stride(1), p.v_sh = v.stride(2);
    p.pk_sb = prefix_k.stride(0), p.pk_ss = prefix_k.stride(1), p.pk_sh = prefix_k.stride(2);
    p.pv_sb = prefix_v.stride(0), p.pv_ss = prefix_v.stride(1), p.pv_sh = prefix_v.stride(2);
    p.B = B, p.Hq = Hq, p.Hkv = Hkv, p.L = L, p.P = P, p.G = G, p.n = n;
    p.np = np, p.no = no, p.prw = prw, p.orw = orw, p.prb = prb, p.orb = orb, p.prefix_blocks = pitems * np;
    p.scale_log2 = softmax_scale * kLog2e;
    if (D == 128) {
      prefix_attend_kernel<E, 128><<<blocks, kThreads, 0, stream>>>(p);
      prefix_join_kernel<E, 128><<<B * Hq, kThreads, 0, stream>>>(p);
    } else {
      prefix_attend_kernel<E, 64><<<blocks, kThreads, 0, stream>>>(p);
      prefix_join_kernel<E, 64><<<B * Hq, kThreads, 0, stream>>>(p);
    }
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return out;
}
