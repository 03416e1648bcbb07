// Fragment, LDS and work-order helpers shared by the attention kernels (flash_attn.hip, shared_attn.hip,
// shared_decode.hip).
#pragma once

#include "dlgm_common.h"

namespace dlgm {

typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __fp16 hf16x4 __attribute__((ext_vector_type(4)));  // the transpose-read builtin's f16 vector type
typedef __attribute__((address_space(3))) hf16x4 lds_f16x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Deferred rescale (forward): the running max used for exponentiation is only raised when a
// row's new max exceeds it by more than 2^kRescaleLog2 -- P stays <= 256, exact in fp32 sums.
constexpr float kRescaleLog2 = 8.f;

// v_exp_f32 as is: exp2f() adds a denormal range fix-up (cmp + cndmask + ldexp per element) that
// softmax does not need (arguments are <= 0 up to the deferred-rescale slack; underflow -> 0).
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Softmax arithmetic on pairs of accumulator registers. The build keeps packed fp32 instructions off, so a pair is two
// scalar instructions (forward 0.575 vs 0.574 ms, backward 1.74 vs 1.76 ms at S 8192, 32/8 heads, D 128: the loops do
// not need the packed forms).
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ f32x2 pk_fma(f32x2 a, f32x2 b, f32x2 c) { return __builtin_elementwise_fma(a, b, c); }

// A condition the caller knows is wave-uniform, made provably so (scalar branch, no exec masking).
__device__ __forceinline__ bool uniform(bool c) { return __builtin_amdgcn_readfirstlane((int)c) != 0; }

__device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// fp16 compute path (DeepSpeed "fp16" block): the same fragment maps on the f16 MFMA
__device__ __forceinline__ f32x16 mfma32(const f16x8& a, const f16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// 16-byte-chunk XOR swizzles (see header). D = head dim, rows of D bf16.
template <int D>
__device__ __forceinline__ int swz_row(int row, int ch) {  // image read by ds_read_b128 rows
  if constexpr (D == 128) return ch ^ (row & 15);
  else if constexpr (D == 32) return ch ^ ((row >> 2) & 3);  // 64-B rows: four rows fill the banks, one image for all
  else return ch ^ ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int swz_tr(int row, int ch) {  // image read by ds_read_b64_tr_b16
  if constexpr (D == 128) return ch ^ ((row & 3) << 2);
  else if constexpr (D == 32) return swz_row<32>(row, ch);
  else return ch ^ (((row >> 1) & 1) << 2);
}
// One image good for both kinds of read (used by the backward's Q / dO / K tiles):
// plain 256-B rows, chunk ^ (((row&3)<<2) | ((row>>2)&3)); the 128-B-row variant
// for D = 64 folds the row parity in instead.
template <int D>
__device__ __forceinline__ int swz_dual(int row, int ch) {
  if constexpr (D == 128) return ch ^ (((row & 3) << 2) | ((row >> 2) & 3));
  else if constexpr (D == 32) return swz_row<32>(row, ch);
  else return ch ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));
}

// Makes x opaque to the optimiser: a per-lane LDS offset computed once before a loop then stays in its
// register instead of being rebuilt from its row and swizzle parts inside the loop (hipcc re-added
// them before every read: one v_add_u32 per ds_read in the backward's tile loops).
__device__ __forceinline__ void pin(int& x) { asm volatile("" : "+v"(x)); }

template <typename E>
__device__ __forceinline__ vec8_t<E> lds_read_b128(const E* base) {
  return *reinterpret_cast<const vec8_t<E>*>(base);
}

// x of lane i ^ 32 (the other half-wave): one v_permlane32_swap instead of an LDS bpermute round trip
__device__ __forceinline__ float swap_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(__lane_id() < 32 ? r[1] : r[0]);
}

// Store one 32-row x D accumulator row block (lane (r, h) holds columns 8k + 4h .. +3 of row r for
// each 8-column group k) as bf16, scaled. One half-exchange (v_permlane32_swap) per dword of a group
// pair (k, k+1) leaves lanes h = 0 with columns 8k .. 8k+7 and lanes h = 1 with 8k+8 .. 8k+15: one
// 16-byte store per pair instead of two 8-byte stores (the tail is store-issue bound). Both lanes of
// a pair share the row, so the swap runs on all lanes and only the store is guarded by `valid`. A row that is not `live`
// (behind a length) is stored as zeros whatever its accumulators hold: 0 times a NaN or an infinity of a live row is a NaN.
template <int DT, typename E>
__device__ __forceinline__ void store_rows_bf16(E* row, const f32x16 (&acc)[DT], float scale, int h, bool valid,
                                                bool live = true) {
#pragma unroll
  for (int k = 0; k < 4 * DT; k += 2) {
    const f32x16& oa = acc[k >> 2];
    const f32x16& ob = acc[(k + 1) >> 2];
    const int ja = 4 * (k & 3), jb = 4 * ((k + 1) & 3);
    vec4_t<E> va = {(E)(oa[ja] * scale), (E)(oa[ja + 1] * scale), (E)(oa[ja + 2] * scale),
                    (E)(oa[ja + 3] * scale)};
    vec4_t<E> vb = {(E)(ob[jb] * scale), (E)(ob[jb + 1] * scale), (E)(ob[jb + 2] * scale),
                    (E)(ob[jb + 3] * scale)};
    uint2 a = __builtin_bit_cast(uint2, va), c = __builtin_bit_cast(uint2, vb);
    const auto sx = __builtin_amdgcn_permlane32_swap(a.x, c.x, false, false);
    const auto sy = __builtin_amdgcn_permlane32_swap(a.y, c.y, false, false);
    if (valid)
      *reinterpret_cast<uint4*>(row + 8 * k + 8 * h) =
          live ? make_uint4(sx[0], sy[0], sx[1], sy[1]) : make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ bf16x4 lds_read_tr(const bf16* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p));
}
__device__ __forceinline__ f16x4 lds_read_tr(const f16* p) {
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_f16x4*)(p)));
}

__device__ __forceinline__ bf16x8 cat(bf16x4 a, bf16x4 b) {
  return (bf16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ f16x8 cat(f16x4 a, f16x4 b) {
  return (f16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

typedef __attribute__((address_space(1))) const void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

// One LDS-DMA piece: 64 lanes x 16 B = 1 KiB landing lane-linearly at `lds` (wave-uniform).
__device__ __forceinline__ void glds16(const void* src, void* lds) {
  __builtin_amdgcn_global_load_lds((gptr_t)src, (lptr_t)lds, 16, 0, 0);
}
__device__ __forceinline__ void glds4(const void* src, void* lds) {
  __builtin_amdgcn_global_load_lds((gptr_t)src, (lptr_t)lds, 4, 0, 0);
}
__device__ __forceinline__ void vm_drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// One LDS-DMA piece through a buffer descriptor (buffer_load_dwordx4 ... lds): `base` and `nbytes`
// are wave-uniform (the descriptor lives in SGPRs, reads at or past nbytes return zero), `voff`
// is the per-lane byte offset, `soff` a wave-uniform byte offset (the tile advance).
__device__ __forceinline__ void dma16(const void* base, int nbytes, uint32_t voff, uint32_t soff, lptr_t lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, nbytes,
                                                                             0x00020000),
                                           lds, 16, voff, soff, 0, 0);
}
__device__ __forceinline__ void dma16(const void* base, int nbytes, uint32_t voff, uint32_t soff, void* lds) {
  dma16(base, nbytes, voff, soff, (lptr_t)const_cast<void*>(lds));
}

// bijective remap of the block id so that consecutive work items land on one XCD
__device__ __forceinline__ int xcd_remap(int id, int total) {
  if (total % 8 != 0) return id;
  return (id % 8) * (total / 8) + id / 8;
}

// LDS-DMA whose arrival only the kernel's own waits (vm_drain) follow. After the builtin the compiler waits for
// every load in flight before the next LDS read that it cannot tell apart from the landing place (any transposed read, any
// buffer chosen at run time): the next tile then loads before, not during, the work on this one -- measured 266 against
// 166 us of work and 156 us of loads alone in the latent attend kernel. An LDS-DMA has no destination register, so nothing
// in flight is known to the register allocator, and its address registers are read when it issues. Every tile is waited
// for and followed by a barrier before it is read, and before the workgroup ends.
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 buffer_of(const void* base, int nbytes) {  // raw buffer: reads at or past nbytes give 0
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return (i32x4){(int)(uint32_t)a, (int)((uint32_t)(a >> 32) & 0xffff), nbytes, 0x00020000};
}
__device__ __forceinline__ uint32_t lds_at(const void* lds) {  // LDS address of a wave-uniform pointer
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lptr_t)const_cast<void*>(lds));
}
// 64 lanes x 16 B (4 B) from base + voff, landing lane-linearly at the wave-uniform LDS address. Two distances the hardware
// does not keep and the compiler does not look for in here: M0 is written 1 wait state before the load or more, and a word of
// the descriptor that a vector instruction wrote (a spilled one comes back by v_readlane) 5 wait states or more. Whatever
// stands in front of the block, the move and s_nop 3 are those 5. (One block for all pieces of a tile, which waits once, is no
// faster: latent attend 232 against 229 us over 32 x 16384 rows, prefix attend 92 against 93 over 16384, dK/dV equal.)
__device__ __forceinline__ void dma16_async(const void* base, int nbytes, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff),
               "s"(buffer_of(base, nbytes)), "s"(lds)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4_async(const void* base, int nbytes, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff),
               "s"(buffer_of(base, nbytes)), "s"(lds)
               : "memory", "m0");
}

// A length given by the caller, cut to what exists; wave-uniform by construction (descriptors are built from it)
__device__ __forceinline__ int clamp_len(int len, int most) {
  return __builtin_amdgcn_readfirstlane(min(max(len, 0), most));
}

// ROWS rows of D elements into an LDS image by LDS-DMA, 1 KiB pieces split over NW waves; the swizzle (0 row, 1 dual,
// 2 transposed-read image) is applied to the source column. `valid` rows exist: the descriptor ends behind the last of
// them and the hardware's bounds check returns zero past it.
template <typename E, int D, int ROWS, int SWZ, int NW = 4>
struct RowTile {
  static constexpr int CH = D / 8, PR = 64 / CH, NP = ROWS / PR, PPW = (NP + NW - 1) / NW;
  static_assert(NP % NW == 0 || NP < NW, "pieces must split evenly over the waves");
  static_assert((NW * PR) % 16 == 0, "piece step must be a multiple of the swizzle period");
  int row, col;  // this lane's row of the first piece, its source byte in the row
  __device__ __forceinline__ RowTile(int wave, int lane) {
    row = wave % NP * PR + lane / CH;
    const int phys = lane % CH;
    col = 16 * (SWZ == 2 ? swz_tr<D>(row, phys) : SWZ == 1 ? swz_dual<D>(row, phys) : swz_row<D>(row, phys));
  }
  __device__ __forceinline__ void issue(E* img, const E* base, int64_t stride, int valid, int wave) const {
    if (NP < NW) wave %= NP;  // fewer pieces than waves: some load one twice, which costs less than a branch
    const int bytes = valid > 0 ? (int)((int64_t)(min(valid, ROWS) - 1) * stride * 2) + D * 2 : 0;
    const uint32_t step = (uint32_t)(stride * 2);
    uint32_t off = (uint32_t)row * step + col;
    const uint32_t lds = lds_at(img + wave * 512);
#pragma unroll
    for (int j = 0; j < PPW; ++j) {
      dma16_async(base, bytes, off, lds + NW * 1024 * j);
      off += NW * PR * step;
    }
  }
};

template <typename E>
__device__ __forceinline__ vec8_t<E> pack8(const f32x16& a, int i) {
  return (vec8_t<E>){(E)a[i + 0], (E)a[i + 1], (E)a[i + 2], (E)a[i + 3],
                     (E)a[i + 4], (E)a[i + 5], (E)a[i + 6], (E)a[i + 7]};
}

// Fragments loaded into registers have arrived here: left to its first use, inside the tile loop, the compiler's wait for
// them would stand in every iteration and there wait for the tiles in flight as well
template <typename V, int N>
__device__ __forceinline__ void settle(V (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// 8 elements of a strided row, zero where !ok
template <typename E>
__device__ __forceinline__ vec8_t<E> row8(const E* p, bool ok) {
  return ok ? *reinterpret_cast<const vec8_t<E>*>(p) : (vec8_t<E>)((E)0.f);
}

// Where a lane reads its fragments in an image of D-wide rows (element offsets). All swizzles XOR the 16-byte chunk of a
// row, whose bits lie below the row's, so every fragment is one lane offset XOR a constant plus an immediate. A loop pins
// the offset once an iteration: left to itself the compiler keeps one register per fragment (some 30 in the wide backward,
// which then spilled 49: dQ 2296 us at S 8192, 32 heads).
template <int D, int SWZ>  // SWZ: 0 row image, 1 dual image
struct RowFrag {           // row `r` of a 32-row block, 8 columns 16 kk + 8 h
  int at;
  __device__ __forceinline__ RowFrag(int r, int h) {
    at = r * D + ((SWZ ? swz_dual<D>(r, h) : swz_row<D>(r, h)) << 3);
  }
  __device__ __forceinline__ int operator()(int kk) const { return at ^ (kk << 4); }
};
template <int D, int SWZ>  // SWZ: 1 dual image, 2 transposed-read image
struct TrFrag {            // columns 32 dt .. +31 of rows row0 + {4 h .. +3, 8 + 4 h .. +3}, transposed: an A operand
  int at;
  __device__ __forceinline__ TrFrag(int h, int i16, int g) {
    const int col = 16 * (g & 1) + 4 * (i16 & 3), row = 4 * h + (i16 >> 2), ch = col >> 3;
    at = row * D + ((SWZ == 2 ? swz_tr<D>(row, ch) : swz_dual<D>(row, ch)) << 3) + (col & 7);
  }
  template <typename E>
  __device__ __forceinline__ vec8_t<E> read(const E* img, int dt, int row0) const {
    constexpr int X = SWZ == 1 || D == 32 ? 16 : 0;  // how the swizzle of row + 8 differs
    const int a = at ^ (dt << 5);
    return cat(lds_read_tr(img + row0 * D + a), lds_read_tr(img + (row0 + 8) * D + (a ^ X)));
  }
};

// fp32 rows of a transposed accumulator: lane (key r, half h) holds columns 8k + 4h .. +3; zeros where not `live`
template <int DT>
__device__ __forceinline__ void store_rows_f32(float* row, const f32x16* acc, float scale, int h, bool live = true) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = {acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
      *reinterpret_cast<f32x4*>(row + dt * 32 + 8 * g + 4 * h) = live ? v * scale : (f32x4)(0.f);
    }
}

// acc = f0 acc + f1 row, rows as store_rows_f32 wrote them
template <int DT>
__device__ __forceinline__ void add_rows_f32(const float* row, f32x16* acc, float f0, float f1, int h) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(row + dt * 32 + 8 * g + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[dt][4 * g + j] = acc[dt][4 * g + j] * f0 + v[j] * f1;
    }
}

}  // namespace dlgm
