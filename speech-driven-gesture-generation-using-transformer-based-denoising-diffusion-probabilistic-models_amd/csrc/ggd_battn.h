// ggd_battn.h -- attention of the training path for any lengths (gfx950): masks, shared kv heads, a
// learned relative position bias, f32 and bf16, forward and backward (include/ggd_train.h,
// ggd_tr_battn_*).
//
//   s_ij = scale q_i . k_j + table[bucket(j - i - offset)][head],  p = softmax over the allowed j
//   o_i  = sum_j p_ij v_j          (a row with no allowed key: o_i = 0, no gradient)
//   delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dq = scale ds k,  dk = scale ds^T q,  dv = p^T do,  dtable[b][head] = sum of ds over the bucket
//
// Every kernel keeps one operand's rows in registers -- lane & 31 = the row -- and streams the other
// side's rows through LDS in tiles.  A product "streamed x stationary" then has the streamed rows
// as the MFMA's M and the stationary row as the lane, so that a stationary row's scores lie in the
// registers of two lanes (l and l ^ 32), the softmax needs one exchange between them, and the
// probabilities are at once the B operand of the next product: its k slots may hold the streamed rows
// in any order, as long as the A operand uses the same one (mma_cols).  Scores stay in registers; weights go through
// LDS from one wave to another in the paired dk / dv kernel alone, and ds on their way into the table's sums by
// diagonals.
//   forward, dq:  stationary = queries (q, do), streamed = keys (k, v)
//   dk, dv:       stationary = keys (k, v),     streamed = queries (q, do)
// dq and dk / dv are two kernels that both form the scores (7 products instead of 5): the sums over
// the streamed side then stay in registers, with no order that varies (the table's sums by distance are LDS adds of
// which no two meet on a word).
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "ggd_common.h"

#include "../../include/ggd_train.h"

namespace ggd {
namespace battn {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;

constexpr int BT_MAX_DK = 128, BT_MAX_DISTANCE = 2047, BT_MAX_BUCKETS = 1024;
constexpr float BT_LOG2E = 1.4426950408889634f;

struct BtArgs : ggd_tr_battn_args {
  int group;       // query heads of a kv head
  int off;         // offset, clamped (past the table's distance on either side all is one bucket)
  int splits;      // parts of the streamed axis
  int fine;        // bf16: weights and ds go into their products with the rest of their rounding too
  int vec_o;       // the written rows take 4-element stores
  int64_t hq, hk;  // elements between the heads of a row of q and dout, of k and v (dk, or what it is padded to)
  int64_t lddo;    // elements between rows of dout
  float c;         // scale log2(e): scores are held in log2 units
  float* part;     // partial results of the splits
  float* delta;    // [n][heads][lq]
  float* dtab;     // partial table gradients [blocks][n_buckets]
  float* rest;     // bf16 with a table gradient: [splits][2][n][heads][lq], what the dq kernel leaves to bt_table_rest_kernel
};

// ---------------------------------------------------------------------------------------------
// LDS images: rows of DK elements in 16-byte units, unit u of row r at u ^ swz(r).  64 banks of 4
// bytes take 16 units at a time.  A row-wise read (lane = row, one unit each) needs 16 consecutive
// rows in different units mod 16; bf16's transposing read (4 rows x 64 bytes) needs the units
// 4 b .. 4 b + 3 of rows 4 a .. 4 a + 3 in different ones; swz is a bijection of the row bits that does both.
// ---------------------------------------------------------------------------------------------
template <typename T, int DK>
struct Img {
  static constexpr int EPU = 16 / sizeof(T), UPR = DK / EPU;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (sizeof(T) == 2) {
      if constexpr (UPR == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
      else if constexpr (UPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
      else return (r >> 2) & 3;
    } else {
      if constexpr (UPR >= 16) return r & 15;
      else return (r >> 1) & 7;
    }
  }
  static __device__ __forceinline__ int unit(int r, int u) { return r * UPR + (u ^ swz(r)); }
};

// rows of a streamed tile: one word of validity bits, one 64-lane load of the mask
template <typename T, int DK>
constexpr int tile_rows() { return sizeof(T) == 4 && DK == 128 ? 32 : 64; }

__device__ __forceinline__ int lane_id() { return threadIdx.x & 63; }

// byte of row r (r + lane) of a mask, or whether the row exists
__device__ __forceinline__ int mask_byte(const uint8_t* mask, int row0, int rows, int count) {
  const int l = lane_id(), r = row0 + l;
  if (l >= rows || r >= count) return 0;
  return mask ? mask[r] : 1;
}

// unit u of a row: zeros past dk.  (Rows are 16-byte aligned and dk whole units: others are packed first.)
template <typename T>
__device__ __forceinline__ uint4 load_unit(const T* __restrict__ row, int u, int dk) {
  constexpr int EPU = 16 / sizeof(T);
  return u * EPU < dk ? *(const uint4*)(row + u * EPU) : make_uint4(0, 0, 0, 0);
}

typedef __attribute__((ext_vector_type(4))) int i32x4;
// a buffer over the memory from a wave-uniform address on; the offset BT_OUT lies past its end and reads as zero
constexpr int BT_OUT = INT32_MIN;
__device__ __forceinline__ i32x4 buffer_at(const void* p) {
  const uint64_t at = (uint64_t)p;
  return i32x4{(int)__builtin_amdgcn_readfirstlane((int)at), (int)(__builtin_amdgcn_readfirstlane((int)(at >> 32)) & 0xFFFF), 0x7FFFFFFF, 0x00020000};
}

__device__ __forceinline__ uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// One tile of rows from memory into an LDS image, straight (buffer loads to LDS: no registers, nothing for the VALU).
// Thread t of 256 (a block's, or its half's) fills unit t + 256 i of the image in instruction i, and reads the row's unit that swz puts there.  Rows whose
// bit is clear are not read: their offset lies past the buffer's end, and zeros go into the image.
//   The loads are issued by asm (the builtin makes the compiler wait for them at the next LDS access); they have
// landed after tile_ready().
template <typename T, int DK, int ROWS>
struct Tile {
  static constexpr int UPR = Img<T, DK>::UPR, N = ROWS * UPR / 256, STEP = 256 / UPR;   // instructions; rows between them
  static_assert(ROWS * UPR % 256 == 0, "whole units a thread");
  static constexpr int KINDS = STEP % 16 ? 2 : 1;   // (f32, 128: rows 8 apart have another swz)
  int row;          // of instruction 0
  int off[KINDS];   // byte offset of its unit, BT_OUT past dk
  __device__ __forceinline__ void start(int64_t ld, int dk) {
    const int t = threadIdx.x & 255;
    row = t / UPR;
#pragma unroll
    for (int k = 0; k < KINDS; ++k) {
      const int u = (t % UPR) ^ Img<T, DK>::swz(row + k * STEP);
      off[k] = u * Img<T, DK>::EPU < dk ? (int)(row * ld * (int64_t)sizeof(T)) + u * 16 : BT_OUT;
    }
  }
  __device__ __forceinline__ void load(const T* base, int64_t ld, uint64_t bits, const uint4* img) const {
    const i32x4 rs = buffer_at(base);
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_at(img) + ((threadIdx.x & 255) >> 6) * 1024);
    const int step = (int)(STEP * ld * (int64_t)sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = off[i % KINDS];
      issue(rs, (bits >> (row + i * STEP)) & 1 && o != BT_OUT ? o + i * step : BT_OUT, at + i * 4096);
    }
  }
  // (five wait states: the descriptor and the address may come from the VALU's readfirstlane.  m0 is given back: it is not a register
  // that asm can declare as written)
  static __device__ __forceinline__ void issue(i32x4 rs, int offset, uint32_t at) {
    uint32_t kept;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(kept) : "s"(at), "v"(offset), "s"(rs) : "memory");
  }
};

// the block's loads have landed in LDS, and every wave is past its last reads of the other buffer
__device__ __forceinline__ void tile_ready() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// the block's LDS writes are there for all of it; loads may still be under way
__device__ __forceinline__ void lds_ready() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// the same through registers, for a wave alone (bt_few_kernel): the loads stay in flight while it works
template <typename T, int DK, int ROWS, int THREADS>
struct Stage {
  static constexpr int UPR = Img<T, DK>::UPR, N = ROWS * UPR / THREADS;
  static_assert(ROWS * UPR % THREADS == 0, "whole units a thread");
  uint4 x[N];
  __device__ __forceinline__ void load(const T* __restrict__ base, int64_t ld, uint64_t bits, int dk, int t) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = t + i * THREADS, r = e / UPR, u = e % UPR;
      x[i] = (bits >> r) & 1 ? load_unit(base + r * ld, u, dk) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void store(uint4* img, int t) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = t + i * THREADS, r = e / UPR, u = e % UPR;
      img[Img<T, DK>::unit(r, u)] = x[i];
    }
  }
};

// ---------------------------------------------------------------------------------------------
// products.  acc: lane & 31 = the stationary row n, register 4 g + j of half h = lane >> 5 holds m = 8 g + 4 h + j
// ---------------------------------------------------------------------------------------------
// a stationary row's elements as B operands: unit 2 s + h of the row (bf16: 8 elements, one 32x32x16
// product; f32: 4 elements, one 32x32x2 product each)
template <typename T, int DK>
struct Frag {
  static constexpr int N = Img<T, DK>::UPR / 2;
  uint4 x[N];
  __device__ __forceinline__ void load(const T* __restrict__ row, int dk, bool there) {
    const int h = lane_id() >> 5;
#pragma unroll
    for (int s = 0; s < N; ++s) x[s] = there ? load_unit(row, 2 * s + h, dk) : make_uint4(0, 0, 0, 0);
  }
  // rows ld apart from `base` on, the same for the wave: zeros come from past the buffer's end, and no load waits for a branch
  __device__ __forceinline__ void load_rows(const T* base, int64_t ld, int dk, bool there) {
    const int l = lane_id(), h = l >> 5, row = (int)((l & 31) * ld * (int64_t)sizeof(T));
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), (short)0, 0x7FFFFFFF, 0x00020000);
#pragma unroll
    for (int s = 0; s < N; ++s)
      x[s] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, there && (2 * s + h) * Img<T, DK>::EPU < dk ? row + (2 * s + h) * 16 : BT_OUT, 0, 0));
  }
};

// acc += rows r0 .. r0 + 31 of the image times the stationary rows (contraction over the elements)
template <typename T, int DK>
__device__ __forceinline__ void mma_rows(f32x16& acc, const uint4* img, int r0, const Frag<T, DK>& b) {
  const int l = lane_id(), r = r0 + (l & 31), h = l >> 5;
#pragma unroll
  for (int s = 0; s < Frag<T, DK>::N; ++s) {
    const uint4 a = img[Img<T, DK>::unit(r, 2 * s + h)];
    if constexpr (sizeof(T) == 2) {
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b.x[s]), acc, 0, 0, 0);
    } else {
      const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b.x[s]);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af[j], bf[j], acc, 0, 0, 0);
    }
  }
}

// acc[mb] += (columns 32 mb .. + 31 of image rows r0 .. r0 + 31)^T times p, p as an acc of those rows.
// bf16: p is rounded to bf16 here (half a step, up to 2^-8 of each weight, on sums that stay in f32); k slot 8 h + i
// of step s is row 16 s + 8 (i / 4) + 4 h + i % 4 -- the rows the half's registers hold -- read by two
// transposing loads.  f32: k slot h of step (g, j) is row 8 g + 4 h + j.
// sum (SUM): + this half's weights as they go into the product, after their rounding
template <typename T, int DK, bool SUM = false>
__device__ __forceinline__ void mma_cols(f32x16 (&acc)[DK / 32], const uint4* img, int r0, const f32x16& p, float* sum = nullptr) {
  const int l = lane_id(), h = l >> 5;
  if constexpr (sizeof(T) == 2) {
    const int i = l & 15, q = i >> 2;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint4 pb = make_uint4(pk_bf16(p[8 * s], p[8 * s + 1]), pk_bf16(p[8 * s + 2], p[8 * s + 3]),
                                  pk_bf16(p[8 * s + 4], p[8 * s + 5]), pk_bf16(p[8 * s + 6], p[8 * s + 7]));
      if constexpr (SUM) {
        typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
        const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3F803F80u);
        const uint32_t w[4] = {pb.x, pb.y, pb.z, pb.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) *sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w[e]), ones, *sum, false);
      }
      const int ra = r0 + 16 * s + 4 * h + q, rb = ra + 8;
#pragma unroll
      for (int mb = 0; mb < DK / 32; ++mb) {
        const int u = 4 * mb + 2 * ((l >> 4) & 1) + ((i & 3) >> 1);
        typedef __attribute__((address_space(3))) bf16x4* lds4;
        const bf16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)((uint2*)(img + Img<T, DK>::unit(ra, u)) + (i & 1)));
        const bf16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)((uint2*)(img + Img<T, DK>::unit(rb, u)) + (i & 1)));
        const bf16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
        acc[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, __builtin_bit_cast(bf16x8, pb), acc[mb], 0, 0, 0);
      }
    }
  } else {
    if constexpr (SUM)
#pragma unroll
      for (int r = 0; r < 16; ++r) *sum += p[r];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + 8 * g + 4 * h + j;
#pragma unroll
        for (int mb = 0; mb < DK / 32; ++mb) {
          const int u = 8 * mb + ((l & 31) >> 2);
          const float a = ((const float*)(img + Img<T, DK>::unit(r, u)))[l & 3];
          acc[mb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[4 * g + j], acc[mb], 0, 0, 0);
        }
      }
  }
}

// what mma_cols' rounding to bf16 leaves of p: a second product of it carries p to 16 bits (BtArgs::fine)
__device__ __forceinline__ f32x16 unrounded(const f32x16& p) {
  f32x16 x;
#pragma unroll
  for (int r = 0; r < 16; r += 2) {
    const uint32_t w = pk_bf16(p[r], p[r + 1]);
    x[r] = p[r] - __uint_as_float(w << 16);
    x[r + 1] = p[r + 1] - __uint_as_float(w & 0xFFFF0000u);
  }
  return x;
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// the other half's value (lane ^ 32) combined with this lane's, the same in both
__device__ __forceinline__ float both_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float both_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// register 4 g + j of this half: row 8 g + 4 h + j of its block of 32
__device__ __forceinline__ int reg_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// whether register r's row has its bit set; w: the block's 32 bits
__device__ __forceinline__ bool row_bit(uint32_t w4, int r) { return (w4 >> (8 * (r >> 2) + (r & 3))) & 1; }   // w4 = w >> 4 h

// a lane's row as it is written: 4 consecutive elements of columns 32 mb + 8 g + 4 h
template <typename T, int DK>
__device__ __forceinline__ void store_row(T* __restrict__ row, const f32x16 (&acc)[DK / 32], float f, int dk, bool vec) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int mb = 0; mb < DK / 32; ++mb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * mb + 8 * g + 4 * h;
      const float v0 = acc[mb][4 * g] * f, v1 = acc[mb][4 * g + 1] * f, v2 = acc[mb][4 * g + 2] * f, v3 = acc[mb][4 * g + 3] * f;
      if (vec) {
        if (c >= dk) continue;
        if constexpr (sizeof(T) == 4) *(f32x4*)(row + c) = f32x4{v0, v1, v2, v3};
        else *(uint2*)(row + c) = make_uint2(pk_bf16(v0, v1), pk_bf16(v2, v3));
      } else {
        if (c < dk) row[c] = from_f32<T>(v0);
        if (c + 1 < dk) row[c + 1] = from_f32<T>(v1);
        if (c + 2 < dk) row[c + 2] = from_f32<T>(v2);
        if (c + 3 < dk) row[c + 3] = from_f32<T>(v3);
      }
    }
}

// ---------------------------------------------------------------------------------------------
// the bias: line[d] of distance d = j - i - offset for -D - 62 .. D + 62, the ends' values past -D and D, in log2 units: a block of
// 32 x 32 places that is not wholly past the table's distance finds each of its places there, and a lane's 16 at
// constant steps from one address.  An entry of -inf forbids
// its places; a finite one past the largest log2 unit counts as that, so that rows of the type's lowest
// value stay a softmax among equals.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float bias_entry(float x) {
  constexpr float most = 2.358e38f;   // largest finite / log2(e)
  return x == -INFINITY ? x : fminf(fmaxf(x, -most), most) * BT_LOG2E + (x != x ? x : 0.f);
}
__device__ __forceinline__ int bucket_of(const BtArgs& a, int d) {   // d in 0 .. 2 D
  return min(max(a.buckets[d], 0), a.n_buckets - 1);
}
constexpr int LINE_PAD = 62;
__device__ __host__ __forceinline__ int line_floats(int D) { return (2 * (D + LINE_PAD) + 1 + 3) / 4 * 4; }
// mem: line_floats(D) floats; line = mem + D + LINE_PAD
__device__ __forceinline__ void bias_line(float* mem, const BtArgs& a, int head) {
  for (int e = threadIdx.x; e <= 2 * (a.distance + LINE_PAD); e += blockDim.x) {
    const int d = min(max(e - LINE_PAD, 0), 2 * a.distance);
    mem[e] = bias_entry(a.table[(int64_t)bucket_of(a, d) * a.heads + head]);
  }
}

// a block of 32 x 32 places whose distances are lo .. hi: all past the table's distance?  They have one bias then.
__device__ __forceinline__ bool past_table(int D, int lo, int hi) { return lo >= D || hi <= -D; }

// ... and one that is worth adding behind the product's scale, in one fma with the maximum (not where it is so large that the
// scores have to vanish beside it, or infinite)
__device__ __forceinline__ bool one_bias(const float* line, int D, int lo, int hi, float& bias) {
  if (!past_table(D, lo, hi)) return false;
  const float b = line[lo >= D ? D : -D];
  if (!(__builtin_amdgcn_readfirstlane(__float_as_int(fabsf(b))) < __float_as_int(4096.f))) return false;
  bias = b;
  return true;
}

// s (raw products) -> log2 units with the bias.  rel: j - i - offset of register row 0 of this half and this lane,
// and sign +1 where the registers run over keys, -1 where they run over queries
template <int SIGN>
__device__ __forceinline__ void add_bias(f32x16& s, const float* line, float c, int rel, int D, int lo, int hi) {
  if (past_table(D, lo, hi)) {
    const float b = line[lo >= D ? D : -D];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, b);
  } else {
    const float* at = line + rel;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, at[SIGN * (8 * (r >> 2) + (r & 3))]);
  }
}

// Sums over the diagonals (equal key - query) of a 32 x 32 block in registers, lane & 31 = query i, register row = key k, into a
// histogram over clamped distances.  16 queries at a time go through an image of the wave's own, [k - i + 15][i], whose
// rows lanes then read: all 32 lanes of the writes and all groups of 16 of the reads are in different banks.  Cells
// without a place stay the zeros of diag_start.  Every lane adds another distance: one order, no two on one word.
constexpr int DIAG = 48 * 20;   // floats of an image
__device__ __forceinline__ void diag_start(float* img) {
  for (int e = lane_id(); e < DIAG; e += 64) img[e] = 0.f;
}
// d0: key 0 - query 0 of the block (with the offset); hist: of distance 0; past, behind: sums at distances >= D, <= -D
__device__ __forceinline__ void diag_add(float* img, float* hist, const f32x16& x, int d0, int D, float& past, float& behind) {
  const int lane = lane_id(), h = lane >> 5, i = lane & 15;
#pragma unroll
  for (int ph = 0; ph < 2; ++ph) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (((lane >> 4) & 1) == ph) {
      float* to = img + 80 * h + 300 - 19 * i;
#pragma unroll
      for (int r = 0; r < 16; ++r) to[20 * (8 * (r >> 2) + (r & 3))] = x[r];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < 47) {
      const f32x4* row = (const f32x4*)(img + 20 * lane);
      const f32x4 a = row[0] + row[1], b = row[2] + row[3], c = a + b;
      const float sum = (c[0] + c[1]) + (c[2] + c[3]);
      const int d = d0 - 16 * ph + lane - 15;
      if (d >= D) past += sum;
      else if (d <= -D) behind += sum;
      else __hip_atomic_fetch_add(hist + d, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
    }
  }
}

// XCD-aware block order: workgroups go to the 8 XCDs in turn.  The `each` items of a clip and kv head (the tiles that share keys
// and values) go to one XCD, so that its L2 holds them once; the clips' kv heads are dealt to the XCDs in turn, so that
// clips of other lengths mix on each.  Where they are few and do not divide, consecutive items go to an XCD.
__host__ __device__ inline bool dealt(uint32_t items, uint32_t each) {
  const uint32_t owners = items / each;
  return owners % 8 == 0 || owners >= 64;
}
__device__ __forceinline__ uint32_t work_item(uint32_t items, uint32_t each) {
  const uint32_t xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
  if (dealt(items, each)) return (xcd + 8 * (at / each)) * each + at % each;
  return xcd * ((items + 7) / 8) + at;
}
inline unsigned work_grid(uint32_t items, uint32_t each) {
  return dealt(items, each) ? (items / each + 7) / 8 * 8 * each : (items + 7) / 8 * 8;
}

struct Launch {
  hipError_t (*pack)(const BtArgs&, const void* src, int64_t ld, int64_t b, int rows, int heads, void* dst, hipStream_t);
  hipError_t (*fwd)(const BtArgs&, hipStream_t);
  hipError_t (*few)(const BtArgs&, hipStream_t);
  hipError_t (*dq)(const BtArgs&, hipStream_t);
  hipError_t (*dkv)(const BtArgs&, hipStream_t);
};

// dynamic LDS past 64 KiB has to be allowed once a device and kernel
template <typename K>
hipError_t allow_lds(K kernel, size_t bytes, std::atomic<bool> (&done)[64]) {
  if (bytes <= 64 * 1024) return hipSuccess;
  int dev = 0;
  if (const hipError_t e = hipGetDevice(&dev)) return e;
  if (dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
    if (const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024)) return e;
    if (dev < 64) done[dev].store(true, std::memory_order_release);
  }
  return hipSuccess;
}

}  // namespace battn
}  // namespace ggd
