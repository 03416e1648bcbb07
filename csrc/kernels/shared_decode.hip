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
// The prefix form is bound by reading the caches once (4 rows D operations to a key). In the latent form a cache row meets
// 2 H (2r + dr) operations: few heads are bound by the cache, 128 by what a tile's steps wait for (31 % of the matrix pipes'
// time, 26 % of the LDS reads', 3.1 TB/s at 32 x 16384 rows). So the work is cut along the length until the chip is full, each sequence by its own length; a part keeps its
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

  __device__ __forceinline__ int len(int b) const { return clamp_len(lens[b], L); }
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
        f = cat(*reinterpret_cast<const vec4_t<E>*>(q + 16 * s + 4 * h),
                *reinterpret_cast<const vec4_t<E>*>(q + 16 * s + 8 + 4 * h));
      acc = mfma32(a[s], f, acc);
    }
    const f32x16 acc1[1] = {acc};
    store_rows_bf16<1>(p.qa + ((int64_t)b * p.H + head) * R + c0 + 32 * w, acc1, 1.f, h, b < p.B);
  }
}

// One workgroup per (sequence, 64 heads, part of its length): tiles of 64 cache rows by LDS-DMA, one ahead (two tiles take
// 72 to 144 KB, one workgroup a CU, so its 8 waves are two a SIMD). Scores, 16x16x32 products: the waves (kq, hb) take 16 rows x 32 heads each over
// all r + dr columns, q in registers (144 at r 512) -- every cache row's LDS reads serve 32 heads, and no wave needs
// another's scores. The weights go through LDS as matrix operands. Outputs, 32x32x16 products: each wave takes r / 8 latent
// columns of all 64 heads. The running reference of a head is raised only when some wave sees it outgrown by
// 2^kRescaleLog2, which all learn at the one barrier between weights and outputs.
constexpr int kLatentThreads = 512;

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// x of lane i ^ 16
__device__ __forceinline__ float swap_quarters(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(__lane_id() & 16 ? r[0] : r[1]);
}

template <typename E, int R, int DR>
__global__ __launch_bounds__(kLatentThreads, 2) void latent_attend_kernel(LatentArgs<E> p) {
  constexpr int NI = R / 128, KR = R / 32, KK = KR + DR / 32;  // images, k-steps of 32 columns
  constexpr int TI = 64 * 128, SLOT = 64 * (R + DR);
  constexpr int DT = R / 256;  // 32-column output tiles of a wave
  __shared__ __attribute__((aligned(16))) E smem[2 * SLOT];
  __shared__ __attribute__((aligned(16))) E pbuf[4][2][512];  // weights: [16 rows][32 heads] fragments of 64 lanes x 8
  __shared__ __attribute__((aligned(16))) E qrope[2][DR / 32][512];  // [32 heads][k-step] fragments of the first 16
  __shared__ float smax[4][64];                              // maxima of 16 rows for 64 heads; at the end, sums
  __shared__ int grown[8];

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5, i16 = lane & 15, g4 = lane >> 4;
  const int kq = w & 3, hb = w >> 2;
  const int nhb = (p.H + 63) / 64;
  // head blocks of one (sequence, part) read the same rows: they follow each other on one XCD
  const int work = xcd_remap(blockIdx.x, gridDim.x);
  const int head0 = work % nhb * 64, part = work / nhb % p.ns, b = work / nhb / p.ns;
  const int len = p.len(b);
  const int tiles = (len + 63) / 64;
  const int t0 = (int)((int64_t)tiles * part / p.ns), t1 = (int)((int64_t)tiles * (part + 1) / p.ns);
  const int blocks = head0 + 32 < p.H ? 2 : 1;  // of 32 heads that exist

  // what a lane derives from its number is derived again for every tile: at r 512 the q fragments and outputs leave no
  // register to keep it in (13 were spilled, and a spilled register's reload waits for the tile in flight as well)
  auto here = [&] {
    int x = lane;
    pin(x);
    return x;
  };
  const E* cb = p.cache + b * p.c_sb;
  auto stage = [&](int buf, int t) {
    const int ln = here();
    const RowTile<E, 128, 64, 1, 8> ct(w, ln);
    const RowTile<E, DR, 64, 0, 8> rt(w, ln);
    E* img = smem + buf * SLOT;
    const E* base = cb + (int64_t)t * 64 * p.c_ss;
#pragma unroll
    for (int i = 0; i < NI; ++i) ct.issue(img + i * TI, base + 128 * i, p.c_ss, len - t * 64, w);
    rt.issue(img + NI * TI, base + R, p.c_ss, len - t * 64, w);
  };
  if (t0 < t1) stage(0, t0);  // on its way beside the q fragments

  vec8_t<E> qf[KK + KR];  // [k-step][16 heads]; the first 16 heads' rope columns stay in LDS, as fragments
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int head = head0 + 32 * hb + 16 * x + i16;
    const E* qa = p.qa + ((int64_t)b * p.H + head) * R + 8 * g4;
    const E* qr = p.q + b * p.q_sb + head * p.q_sh + p.dn + 8 * g4;
#pragma unroll
    for (int kk = 0; kk < KR; ++kk) qf[2 * kk + x] = row8(qa + 32 * kk, head < p.H);
#pragma unroll
    for (int kk = 0; kk < KK - KR; ++kk) {
      const vec8_t<E> f = row8(qr + 32 * kk, head < p.H);
      if (x) qf[2 * KR + kk] = f;
      else *reinterpret_cast<vec8_t<E>*>(&qrope[hb][kk][8 * lane]) = f;  // the same from each of the block's four waves
    }
  }
  settle(qf);
  f32x16 o[2][DT];  // [head block][column tile]
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = (f32x16)(0.f);
  // references (log2 domain) of the heads of this lane's scores, 16 x + i16 of block hb, and of its outputs, 32 x + r
  float m_s[2] = {-INFINITY, -INFINITY}, m_o[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  for (int t = t0, buf = 0; t < t1; ++t, buf ^= 1) {
    vm_drain();
    __syncthreads();
    if (t + 1 < t1) stage(buf ^ 1, t + 1);
    const E* img = smem + buf * SLOT;
    f32x4 s[2] = {(f32x4)(0.f), (f32x4)(0.f)};
    if (hb < blocks) {
      // rows of this wave, columns 8 g4 of a 32-column step
      const int ln = here(), row = 16 * kq + (ln & 15);
      const int ca = row * 128 + (swz_dual<128>(row, ln >> 4) << 3), ra = NI * TI + row * DR + (swz_row<DR>(row, ln >> 4) << 3);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const vec8_t<E> a = lds_read_b128(img + (kk < KR ? kk / 4 * TI + (ca ^ (kk % 4 << 5)) : (ra ^ (kk - KR << 5))));
        s[0] = mfma16(a, kk < KR ? qf[2 * kk] : lds_read_b128(&qrope[hb][kk - KR][8 * ln]), s[0]);
        s[1] = mfma16(a, kk < KR ? qf[2 * kk + 1] : qf[KR + kk], s[1]);
      }
    }
    if (uniform(t * 64 + 64 > len)) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t * 64 + 16 * kq + 4 * g4 + j >= len) s[0][j] = s[1][j] = -INFINITY;
    }
    float mx[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) mx[x] = fmaxf(fmaxf(s[x][0], s[x][1]), fmaxf(s[x][2], s[x][3])) * p.scale_log2;
    // weights over the references so far: right unless a head outgrew its own, which is seen at the barrier
    float sum[2];
    auto weigh = [&] {
      const int ln = here(), q4 = ln >> 4;
      E* to = &pbuf[kq][hb][((ln & 15) + 32 * (q4 & 1)) * 8 + 4 * (q4 >> 1)];  // rows 4 g4 .. +3 of head i16
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float m = m_s[x] == -INFINITY ? 0.f : m_s[x];
        f32x4 e;
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = fast_exp2(s[x][j] * p.scale_log2 - m);
        sum[x] = (e[0] + e[1]) + (e[2] + e[3]);
        *reinterpret_cast<vec4_t<E>*>(to + 16 * x * 8) = __builtin_convertvector(e, vec4_t<E>);
      }
    };
    weigh();
    const int big = __any(mx[0] > m_s[0] + kRescaleLog2 || mx[1] > m_s[1] + kRescaleLog2);
    if (lane == 0) grown[w] = big;
    __syncthreads();
    if (__any(grown[lane & 7] != 0)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        mx[x] = fmaxf(mx[x], swap_quarters(mx[x]));
        mx[x] = fmaxf(mx[x], swap_halves(mx[x]));
        if (g4 == 0) smax[kq][32 * hb + 16 * x + i16] = mx[x];
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int hs = 32 * hb + 16 * x + i16, ho = 32 * x + r;
        const float ns = fmaxf(m_s[x], fmaxf(fmaxf(smax[0][hs], smax[1][hs]), fmaxf(smax[2][hs], smax[3][hs])));
        const float no = fmaxf(m_o[x], fmaxf(fmaxf(smax[0][ho], smax[1][ho]), fmaxf(smax[2][ho], smax[3][ho])));
        l_run[x] *= ns == -INFINITY ? 1.f : fast_exp2(m_s[x] - ns);
        const float alpha = no == -INFINITY ? 1.f : fast_exp2(m_o[x] - no);
        m_s[x] = ns, m_o[x] = no;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= alpha;
      }
      weigh();
      __syncthreads();
    }
    l_run[0] += sum[0], l_run[1] += sum[1];
    const int ln = here();
    const TrFrag<128, 1> vf(ln >> 5, ln & 15, ln >> 4);
    // 16 rows a step: their weights for both head blocks, and this wave's columns of them
    vec8_t<E> pf[4][2], vv[4][DT];
    auto load = [&](int k) {
      if (k >= 4) return;
#pragma unroll
      for (int x = 0; x < 2; ++x) pf[k][x] = lds_read_b128(&pbuf[k][x][8 * ln]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int col = w * DT + dt;  // 32-column tile of the latent vector
        TrFrag<128, 1> vc = vf;
        vc.at ^= (col % 4) << 5;
        vv[k][dt] = vc.read(img + col / 4 * TI, 0, 16 * k);
      }
    };
    load(0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      load(k + 1);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int x = 0; x < 2; ++x) o[x][dt] = mfma32(vv[k][dt], pf[k][x], o[x][dt]);
      __builtin_amdgcn_sched_barrier(0);  // no more fragments in flight than there are registers
    }
  }

  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float l = l_run[x] + swap_quarters(l_run[x]);
    l += swap_halves(l);
    if (g4 == 0) smax[kq][32 * hb + 16 * x + i16] = l;
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int hd = head0 + 32 * x + r;
    if (hd >= p.H) continue;
    const int64_t slot = ((int64_t)b * p.H + hd) * p.ns + part;
    if (w == 0 && h == 0) {
      p.ml[2 * slot] = m_o[x];
      p.ml[2 * slot + 1] = (smax[0][32 * x + r] + smax[1][32 * x + r]) + (smax[2][32 * x + r] + smax[3][32 * x + r]);
    }
    if (t0 < t1) store_rows_f32<DT>(p.o + slot * R + w * DT * 32, o[x], 1.f, h);  // an empty part is not read
  }
}

// One workgroup per (head, 8 sequences): join the parts into the latent outputs, then out = W_v[h] o. What another XCD has
// just written takes some 3 us to arrive (measured: one more round of part loads adds that), so everything is asked for at
// once: every wave takes one sequence's parts, or, for few sequences, a share of them, and its piece of W_v. The latent
// output enters its product as two 16-bit terms (value and remainder), so it is not rounded: the product is a small part
// of the call.
constexpr int kProjectRows = 8, kProjectThreads = 512;
template <typename E, int R, int DV>
__global__ __launch_bounds__(kProjectThreads) void latent_project_kernel(LatentArgs<E> p) {
  constexpr int LD = R + 8, TILES = DV / 32, KP = 8 / TILES, KS = R / 16 / KP;  // column tiles, shares of r, k-steps of one
  constexpr int BATCH = 8;  // parts in flight
  __shared__ __attribute__((aligned(16))) float red[8][R];  // by wave; then the products' shares
  __shared__ __attribute__((aligned(16))) E ol[2][kProjectRows * LD];
  static_assert(8 * 2 * 8 * 16 <= 8 * R, "the shares fit");
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int work = xcd_remap(blockIdx.x, gridDim.x), nb = (p.B + kProjectRows - 1) / kProjectRows;
  const int head = work / nb, b0 = work % nb * kProjectRows;  // workgroups of one head read the same W_v
  const int rows = min(kProjectRows, p.B - b0);
  const int lg = rows > 4 ? 3 : rows > 2 ? 2 : rows > 1 ? 1 : 0, share = 8 >> lg;  // waves of a sequence
  const int seq = min(w >> (3 - lg), rows - 1), first = w & (share - 1);  // waves past the batch repeat its last sequence

  const int64_t slot = ((int64_t)(b0 + seq) * p.H + head) * p.ns;
  const float* ml = p.ml + 2 * slot;
  const int col = lane * 8 % R;  // r 256: the upper lanes repeat the lower
  const float* o = p.o + slot * R + col;
  f32x8 x[BATCH], acc = (f32x8)(0.f);
  auto load = [&](int s0) {
#pragma unroll
    for (int s = 0; s < BATCH; ++s) x[s] = load8(o + min(s0 + s * share, p.ns - 1) * R);
  };
  load(first);
  const int tile = w % TILES, k0 = w / TILES * KS;
  const E* wv = p.w + ((int64_t)head * (p.dn + p.dv) + p.dn + 32 * tile + r) * p.w_ss + 16 * k0 + 8 * h;
  vec8_t<E> wf[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) wf[kk] = *reinterpret_cast<const vec8_t<E>*>(wv + 16 * kk);
  float m = -INFINITY, l = 0.f;  // of the sequence, the same in every lane
#pragma unroll 8
  for (int s = 0; s < p.ns; ++s) m = fmaxf(m, ml[2 * s]);
#pragma unroll 8
  for (int s = 0; s < p.ns; ++s) l += ml[2 * s + 1] == 0.f ? 0.f : fast_exp2(ml[2 * s] - m) * ml[2 * s + 1];
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a sequence without keys: zeros
  for (int s0 = first; s0 < p.ns; s0 += BATCH * share) {
    if (s0 > first) load(s0);
#pragma unroll
    for (int s = 0; s < BATCH; ++s) {
      const int k = s0 + s * share, kc = min(k, p.ns - 1);
      // an empty part (a NaN sum is none): nothing was written there
      const float f = k < p.ns && ml[2 * kc + 1] != 0.f ? fast_exp2(ml[2 * kc] - m) * inv : 0.f;
      acc += f == 0.f ? (f32x8)(0.f) : x[s] * f;
    }
  }
  *reinterpret_cast<f32x8*>(&red[w][col]) = acc;
  __syncthreads();
  for (int i = threadIdx.x * 8; i < rows * R; i += kProjectThreads * 8) {
    const int k = i / R, c = i % R;
    f32x8 v = load8(&red[k * share][c]);
    for (int j = 1; j < share; ++j) v += load8(&red[k * share + j][c]);
    const vec8_t<E> hi = __builtin_convertvector(v, vec8_t<E>);
    *reinterpret_cast<vec8_t<E>*>(ol[0] + k * LD + c) = hi;
    store8f(ol[1] + k * LD + c, v - __builtin_convertvector(hi, f32x8));
  }
  __syncthreads();
  const int at = r % kProjectRows * LD + 16 * k0 + 8 * h;  // columns past the sequences are not stored
  f32x16 out[2] = {(f32x16)(0.f), (f32x16)(0.f)};
#pragma unroll
  for (int kk = 0; kk < KS; ++kk)
#pragma unroll
    for (int y = 0; y < 2; ++y) out[y] = mfma32(wf[kk], lds_read_b128(ol[y] + at + 16 * kk), out[y]);
  out[0] += out[1];
  float* mine = &red[0][0] + ((w * 2 + h) * 8 + r) * 16;  // red has been read
  if (r < 8) {
#pragma unroll
    for (int j = 0; j < 16; j += 8)
      *reinterpret_cast<f32x8*>(mine + j) = (f32x8){out[0][j], out[0][j + 1], out[0][j + 2], out[0][j + 3],
                                                    out[0][j + 4], out[0][j + 5], out[0][j + 6], out[0][j + 7]};
  }
  __syncthreads();
  if (w >= TILES) return;
  f32x16 sum[1] = {(f32x16)(0.f)};
  for (int k = 0; k < KP; ++k) {
    const float* from = &red[0][0] + (((w + k * TILES) * 2 + h) * 8 + r % 8) * 16;
#pragma unroll
    for (int j = 0; j < 16; ++j) sum[0][j] += from[j];
  }
  store_rows_bf16<1>(p.out + ((int64_t)(b0 + r) * p.H + head) * DV + 32 * w, sum, 1.f, h, r < rows);
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

// One workgroup per (kv head, block of rows, part of a key range): 64 keys a step by LDS-DMA, one step ahead, two workgroups
// a CU. The rows are (sequence of the group, q head of the kv head) for the prefix and the q heads for a sequence's own
// keys. rw of the 4 waves stand along the rows: 128 rows take a step's keys whole, 64 share its two halves between pairs of
// waves, 32 between two waves -- few rows are bound by the cache alone, which all 4 waves load.
constexpr int kStep = 64;
template <typename E, int D>
__global__ __launch_bounds__(kThreads, 2) void prefix_attend_kernel(PrefixArgs<E> p) {
  constexpr int KK = D / 16, DT = D / 32;
  constexpr int TI = kStep * D, SLOT = 2 * TI;
  __shared__ __attribute__((aligned(16))) E smem[2 * SLOT];
  __shared__ float sm[4][32], sl[4][32];
  static_assert(sizeof(E) * 2 * SLOT == 4 * 32 * D * 4, "the rows of four waves fit the tiles' space");

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
    len = p.plens ? clamp_len(p.plens[g], p.P) : p.P;
    kb = p.pk + g * p.pk_sb + hk * p.pk_sh, vb = p.pv + g * p.pv_sb + hk * p.pv_sh;
    k_ss = p.pk_ss, v_ss = p.pv_ss;
  } else {
    int x = xcd_remap(blockIdx.x - p.prefix_blocks, gridDim.x - p.prefix_blocks);
    rw = p.orw, nparts = p.no;
    rb = x % p.orb, x /= p.orb;
    part = x % p.no, x /= p.no;
    hk = x % p.Hkv;
    b0 = x / p.Hkv, nrows = rep;
    len = clamp_len(p.lens[b0], p.L);
    kb = p.k + b0 * p.k_sb + hk * p.k_sh, vb = p.v + b0 * p.v_sb + hk * p.v_sh;
    k_ss = p.k_ss, v_ss = p.v_ss;
  }
  const int kw = w / rw;  // which half of a step's keys, where the rows leave waves to share them (others: none)
  const int idx = (rb * rw + w % rw) * 32 + r, seq = b0 + idx / rep, hq = hk * rep + idx % rep;
  const bool ok = idx < nrows;
  const int steps = (len + kStep - 1) / kStep;
  const int t0 = (int)((int64_t)steps * part / nparts), t1 = (int)((int64_t)steps * (part + 1) / nparts);

  const RowTile<E, D, kStep, 0> kt(w, lane);
  const RowTile<E, D, kStep, 2> vt(w, lane);
  auto stage = [&](int buf, int t) {
    E* img = smem + buf * SLOT;
    kt.issue(img, kb + (int64_t)t * kStep * k_ss, k_ss, len - t * kStep, w);
    vt.issue(img + TI, vb + (int64_t)t * kStep * v_ss, v_ss, len - t * kStep, w);
  };
  if (t0 < t1) stage(0, t0);  // on its way beside the q fragments
  vec8_t<E> qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qf[kk] = row8(p.q + seq * p.q_sb + hq * p.q_sh + 16 * kk + 8 * h, ok);
  settle(qf);
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = (f32x16)(0.f);
  float m_run = -INFINITY, l_run = 0.f;
  const RowFrag<D, 0> kf(r, h);
  const TrFrag<D, 2> vf(h, i16, g4);
  // U blocks of 32 keys from image rows ki on, the first of them key0
  auto blocks = [&](auto uc, const E* ki, int key0) {
    constexpr int U = decltype(uc)::value;
    const E* vi = ki + TI;
    f32x16 s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = (f32x16)(0.f);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int u = 0; u < U; ++u) s[u] = mfma32(lds_read_b128(ki + 32 * u * D + kf(kk)), qf[kk], s[u]);
    if (uniform(key0 + 32 * U > len)) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (key0 + 32 * u + (i & 3) + 8 * (i >> 2) + 4 * h >= len) s[u][i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
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
    vec8_t<E> pf[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = fast_exp2(s[u][i] * p.scale_log2 - m_use);
        l_run += s[u][i];
      }
      pf[u][0] = pack8<E>(s[u], 0), pf[u][1] = pack8<E>(s[u], 8);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) o[dt] = mfma32(vf.read(vi, dt, 32 * u + 16 * s2), pf[u][s2], o[dt]);
  };
  for (int t = t0; t < t1; ++t) {
    vm_drain();
    __syncthreads();
    const int buf = (t - t0) & 1;
    if (t + 1 < t1) stage(buf ^ 1, t + 1);
    const E* ki = smem + buf * SLOT;
    const int key0 = t * kStep + 32 * kw;
    if (rw == 4) blocks(std::integral_constant<int, 2>{}, ki, key0);
    else if (kw < 2 && key0 < len) blocks(std::integral_constant<int, 1>{}, ki + 32 * kw * D, key0);
  }

  const int slots = p.np + p.no, slot = pre ? part : p.np + part;
  const float l = l_run + swap_halves(l_run);
  if (rw == 4) {  // no other wave has these rows
    if (ok) {
      const int64_t at = ((int64_t)seq * p.Hq + hq) * slots + slot;
      if (h == 0) p.ml[2 * at] = m_run, p.ml[2 * at + 1] = l;
      if (t0 < t1) store_rows_f32<DT>(p.o + at * D, o, 1.f, h);  // an empty part is not read
    }
    return;
  }
  if (h == 0) sm[w][r] = m_run, sl[w][r] = l;
  __syncthreads();  // also: the last tiles have been read
  const float m = fmaxf(sm[w % rw][r], sm[w % rw + rw][r]);
  const float f = l == 0.f ? 0.f : fast_exp2(m_run - m);
  float* joined = reinterpret_cast<float*>(smem);  // rows of D floats, each turned by 4 per row so that no bank repeats
  if (kw < 2) {
    float* row = joined + (w * 32 + r) * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = {o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
        *reinterpret_cast<f32x4*>(row + ((dt * 32 + 8 * g + 4 * h + 4 * r) & (D - 1))) = v * f;
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rw * 32 * (D / 4); i += kThreads) {
    const int row = i / (D / 4), c = i % (D / 4) * 4, x = row >> 5, rr = row & 31;
    const int id = (rb * rw + x) * 32 + rr;
    if (id >= nrows) break;
    const int64_t a = ((int64_t)(b0 + id / rep) * p.Hq + hk * rep + id % rep) * slots + slot;
    const int turned = (c + 4 * rr) & (D - 1);
    if (c == 0) {
      const float m0 = sm[x][rr], m1 = sm[x + rw][rr], l0 = sl[x][rr], l1 = sl[x + rw][rr], mm = fmaxf(m0, m1);
      p.ml[2 * a] = mm;
      p.ml[2 * a + 1] = (l0 == 0.f ? 0.f : l0 * fast_exp2(m0 - mm)) + (l1 == 0.f ? 0.f : l1 * fast_exp2(m1 - mm));
    }
    if (t0 < t1)
      *reinterpret_cast<f32x4*>(p.o + a * D + c) = *reinterpret_cast<const f32x4*>(joined + row * D + turned) +
                                                    *reinterpret_cast<const f32x4*>(joined + (row + rw * 32) * D + turned);
  }
}

// One workgroup per (sequence, q head): its waves take the parts in turn, then the four sums are added.
template <typename E, int D>
__global__ __launch_bounds__(kThreads) void prefix_join_kernel(PrefixArgs<E> p) {
  constexpr int V = D / 64;  // columns of a lane
  __shared__ float red[4][D];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slots = p.np + p.no;  // at most 128
  const int64_t row = blockIdx.x, base = row * slots;
  float ms[2] = {-INFINITY, -INFINITY}, ls[2] = {0.f, 0.f}, l = 0.f, acc[V] = {};
#pragma unroll
  for (int x = 0; x < 2; ++x)
    if (64 * x + lane < slots) ms[x] = p.ml[2 * (base + 64 * x + lane)], ls[x] = p.ml[2 * (base + 64 * x + lane) + 1];
  const float m = wave_max(fmaxf(ms[0], ms[1]));
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float f = ls[x] == 0.f ? 0.f : fast_exp2(ms[x] - m);  // an empty part (a NaN sum is none)
    l += f * ls[x];
#pragma unroll 8
    for (int s = 64 * x + w; s < min(slots, 64 * x + 64); s += 4) {  // loads without a branch: eight in flight
      const float fs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s & 63));
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = p.o[(base + s) * D + lane * V + j];
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += fs == 0.f ? 0.f : fs * o[j];  // nothing was written to an empty part
    }
  }
  l = wave_sum(l);
#pragma unroll
  for (int j = 0; j < V; ++j) red[w][lane * V + j] = acc[j];
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int c = threadIdx.x;
  const float o = red[0][c] + red[1][c] + red[2][c] + red[3][c];
  p.out[row * D + c] = (E)(l == 0.f ? 0.f : o / l);  // a row without keys: zeros
}

constexpr int64_t kMostParts = 64;  // a join reads every part of a row

// Latent attend: how many parts `items` lengths of `steps` tiles are cut into. A CU holds one workgroup, so the call takes
// (rounds of 256 workgroups) x (tiles of a part + what a workgroup's start and end cost, some 6 tiles); the fewest that make
// that least. (As many as give 256 workgroups or a few more, rounded up, measured 87 us at 5 x 9000 rows, 128 heads, 87 at
// 40 x 2000, 64 heads, and 178 at 96 x 3000; so 57, 66 and 138.)
int64_t latent_parts(int64_t steps, int64_t items) {
  int64_t best = INT64_MAX, ns = 1;
  for (int64_t k = 1; k <= std::min(kMostParts, steps); ++k) {
    const int64_t cost = (items * k + 255) / 256 * ((steps + k - 1) / k + 6);
    if (cost < best) best = cost, ns = k;
  }
  return ns;
}

// waves along the rows: as many as the rows fill (a step's keys are shared by the rest). 256 rows over 16384 keys: 94 us of
// attend with 4, 110 with 2, 153 with 1; 16 rows over 8192: the call 22.8, 21.7 and 21.7.
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
  const int64_t ns = latent_parts((L + 63) / 64, B * nhb);
  auto qa = at::empty({B, H, r}, q.options());
  auto o = at::empty({B, H, ns, r}, q.options().dtype(at::kFloat));
  auto ml = at::empty({B, H, ns, 2}, q.options().dtype(at::kFloat));
  const int64_t a_blocks = check_blocks(H * (r / 128), op), t_blocks = check_blocks(2 * B * nhb * ns, op) / 2;
  const int64_t p_blocks = check_blocks(2 * H * ((B + kProjectRows - 1) / kProjectRows), op) / 2;
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    LatentArgs<E> p{};
    p.q = ptr<E>(q), p.cache = ptr<E>(cache), p.w = ptr<E>(w_kv), p.qa = ptr<E>(qa), p.out = ptr<E>(out);
    p.o = o.data_ptr<float>(), p.ml = ml.data_ptr<float>(), p.lens = lp;
    p.q_sb = stride_of(q, 0), p.q_sh = stride_of(q, 1), p.w_ss = stride_of(w_kv, 0);
    p.c_sb = stride_of(cache, 0), p.c_ss = stride_of(cache, 1);
    p.B = B, p.H = H, p.L = L, p.dn = dn, p.dv = dv, p.ns = ns;
    p.scale_log2 = softmax_scale * kLog2e;
    auto run = [&](auto rc) {
      constexpr int R = decltype(rc)::value;
      if (dn == 128) {
        latent_absorb_kernel<E, 128><<<a_blocks, kThreads, 0, stream>>>(p, R);
        latent_attend_kernel<E, R, 64><<<t_blocks, kLatentThreads, 0, stream>>>(p);
        latent_project_kernel<E, R, 128><<<p_blocks, kProjectThreads, 0, stream>>>(p);
      } else {
        latent_absorb_kernel<E, 64><<<a_blocks, kThreads, 0, stream>>>(p, R);
        latent_attend_kernel<E, R, 32><<<t_blocks, kLatentThreads, 0, stream>>>(p);
        latent_project_kernel<E, R, 64><<<p_blocks, kProjectThreads, 0, stream>>>(p);
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
  const int64_t rep = Hq / Hkv, n = B / G, psteps = (P + kStep - 1) / kStep, osteps = (L + kStep - 1) / kStep;
  const int prw = row_waves(n * rep), orw = row_waves(rep);
  const int64_t prb = (n * rep + 32 * prw - 1) / (32 * prw), orb = (rep + 32 * orw - 1) / (32 * orw);
  // both kinds of workgroup get about the same number of steps, 512 workgroups in all: two a CU, all at once. Where rounding
  // up the parts gives a few more, which would wait for a second round, parts up to half as long again are taken if they
  // end that (16 x 700 keys over 8000, 32/8 heads: 26.7 and 22.7 us); longer ones cost more than the round (96 x 256 over
  // 8192, 64/4 heads, where they would be four times as long: 52 and 99).
  const int64_t pitems = G * Hkv * prb, oitems = B * Hkv * orb;
  auto parts = [](int64_t steps, int64_t per) { return std::min(kMostParts, (steps + per - 1) / per); };
  int64_t per = std::max<int64_t>(1, (pitems * psteps + oitems * osteps + 511) / 512);
  auto fits = [&](int64_t x) { return pitems * parts(psteps, x) + oitems * parts(osteps, x) <= 512; };
  for (int64_t x = per, most = per + (per + 1) / 2; x <= most; x += 1 + x / 16)
    if (fits(x)) {
      per = x;
      break;
    }
  const int64_t np = parts(psteps, per), no = parts(osteps, per);
  if (np + no == 0) return out.zero_();
  auto o = at::empty({B, Hq, np + no, D}, q.options().dtype(at::kFloat));
  auto ml = at::empty({B, Hq, np + no, 2}, q.options().dtype(at::kFloat));
  const int64_t blocks = check_blocks(pitems * np + oitems * no, op), rows = check_blocks(B * Hq, op);
  auto stream = c10::hip::getCurrentHIPStream();
  DLGM_DISPATCH_16(q.scalar_type(), E, {
    PrefixArgs<E> p{};
    p.q = ptr<E>(q), p.k = ptr<E>(k), p.v = ptr<E>(v), p.pk = ptr<E>(prefix_k), p.pv = ptr<E>(prefix_v), p.out = ptr<E>(out);
    p.o = o.data_ptr<float>(), p.ml = ml.data_ptr<float>(), p.lens = lp, p.plens = pp;
    p.q_sb = stride_of(q, 0), p.q_sh = stride_of(q, 1);
    p.k_sb = stride_of(k, 0), p.k_ss = stride_of(k, 1), p.k_sh = stride_of(k, 2);
    p.v_sb = stride_of(v, 0), p.v_ss = stride_of(v, 1), p.v_sh = stride_of(v, 2);
    p.pk_sb = stride_of(prefix_k, 0), p.pk_ss = stride_of(prefix_k, 1), p.pk_sh = stride_of(prefix_k, 2);
    p.pv_sb = stride_of(prefix_v, 0), p.pv_ss = stride_of(prefix_v, 1), p.pv_sh = stride_of(prefix_v, 2);
    p.B = B, p.Hq = Hq, p.Hkv = Hkv, p.L = L, p.P = P, p.G = G, p.n = n;
    p.np = np, p.no = no, p.prw = prw, p.orw = orw, p.prb = prb, p.orb = orb, p.prefix_blocks = pitems * np;
    p.scale_log2 = softmax_scale * kLog2e;
    if (D == 128) {
      prefix_attend_kernel<E, 128><<<blocks, kThreads, 0, stream>>>(p);
      prefix_join_kernel<E, 128><<<rows, kThreads, 0, stream>>>(p);
    } else {
      prefix_attend_kernel<E, 64><<<blocks, kThreads, 0, stream>>>(p);
      prefix_join_kernel<E, 64><<<rows, kThreads, 0, stream>>>(p);
    }
  });
  DLGM_CHECK_HIP(hipGetLastError());
  return out;
}
