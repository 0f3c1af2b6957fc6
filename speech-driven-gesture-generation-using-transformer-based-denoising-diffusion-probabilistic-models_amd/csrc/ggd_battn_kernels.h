// ggd_battn_kernels.h -- the kernels of ggd_battn.h for one element type (included by ggd_battn*.hip)
#pragma once
#include <type_traits>

#include "ggd_battn.h"

namespace ggd {
namespace battn {

// Waves a SIMD in the kernels' launch bounds: 2 where the registers allow it (256 each).  The compiler then keeps the products'
// results in VGPRs, where the VALU works on them; with 1 it gives the sums AGPRs, 256 more, and moves the scores.
constexpr int BT_ROWS = 128;   // stationary rows of a block of the tiled kernels: 4 waves of 32

// ---------------------------------------------------------------------------------------------
// Running softmax of the lane's query over blocks of 32 keys.  m only follows the blocks' maximum when that
// passes it by more than 8 (log2 units): weights then reach 2^8 at most and o is rescaled a few times
// in all instead of in every block.
// ---------------------------------------------------------------------------------------------
template <int DK>
struct Softmax {
  float m, l, lr;   // sums over this half's keys (l: where it is kept, for the backward pass)
  f32x16 o[DK / 32];
  __device__ __forceinline__ void start() {
    m = -INFINITY;
    l = lr = 0.f;
#pragma unroll
    for (int mb = 0; mb < DK / 32; ++mb) o[mb] = zero16();
  }
  // this half's sums -> the row's; f32 rounds no weight, and has one sum
  template <typename T>
  __device__ __forceinline__ void finish() {
    lr = both_sum(lr);
    l = sizeof(T) == 4 ? lr : both_sum(l);
  }
  __device__ __forceinline__ void raise(float mt) {   // mt: the blocks' maximum, the same in both halves
    if (__any(mt > m + 8.f)) {
      const float mn = fmaxf(m, mt), f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
      for (int mb = 0; mb < DK / 32; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[mb][r] *= f;
      l *= f;
      lr *= f;
      m = mn;
    }
  }
};

__device__ __forceinline__ float max16(const f32x16& s) {
  float a = fmaxf(fmaxf(s[0], s[1]), s[2]), b = fmaxf(fmaxf(s[3], s[4]), s[5]);
  float c = fmaxf(fmaxf(s[6], s[7]), s[8]), d = fmaxf(fmaxf(s[9], s[10]), s[11]);
  a = fmaxf(fmaxf(a, s[12]), s[13]);
  b = fmaxf(fmaxf(b, s[14]), s[15]);
  return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// scores of NB blocks of 32 keys against the lane's query -> weights, the running softmax moved on
// rel: (first key) + 4 h - (query position); q0: least query position of the wave
template <typename T, int DK, bool BIAS, int NB>
__device__ __forceinline__ void attend(Softmax<DK>& sm, const uint4* kimg, const uint4* vimg, const Frag<T, DK>& q,
                                       uint64_t bits, const BtArgs& a, const float* line, int rel, int lo, int hi) {
  const int h = lane_id() >> 5;
  f32x16 s[NB];
  float mt = -INFINITY, f[NB], e[NB];   // scores in log2 units: f s + e
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    s[b] = zero16();
    mma_rows<T, DK>(s[b], kimg, 32 * b, q);
    f[b] = a.c;
    e[b] = 0.f;
    if constexpr (BIAS) {
      const int D = a.distance;
      if (!one_bias(line, D, lo + 32 * b, hi + 32 * b, e[b])) {
        add_bias<1>(s[b], line, a.c, rel + 32 * b, D, lo + 32 * b, hi + 32 * b);
        f[b] = 1.f;
      }
    }
    const uint32_t w = (uint32_t)(bits >> (32 * b));
    if (w != 0xFFFFFFFFu) {
      const uint32_t w4 = w >> (4 * h);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = row_bit(w4, r) ? s[b][r] : -INFINITY;
    }
    mt = fmaxf(mt, fmaf(max16(s[b]), f[b], e[b]));
  }
  sm.raise(both_max(mt));
  const float m = sm.m == -INFINITY ? 0.f : sm.m;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    e[b] -= m;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], f[b], e[b]));
    if (sizeof(T) == 2 && a.stat) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sm.l += s[b][r];
    }
    mma_cols<T, DK, true>(sm.o, vimg, 32 * b, s[b], &sm.lr);
    if (sizeof(T) == 2 && a.fine) mma_cols<T, DK, true>(sm.o, vimg, 32 * b, unrounded(s[b]), &sm.lr);
  }
}

// ---------------------------------------------------------------------------------------------
// forward, many rows: a block per 128 query rows of one head; the waves share the key tiles.  32 rows a wave fill the
// MFMA's N, and a tile of 64 keys in LDS (two: the next one arrives by LDS loads meanwhile) serves 4 of them.  Where blocks are
// few the keys are divided too, and bt_join_kernel joins the parts.
//   Bound by the VALU and the MFMA units, which two waves a SIMD overlap in part: exp, maximum and sum of a score are 4 VALU
// operations a lane, and at dk = 64 take more time than its products (counters, of the cycles a kernel runs: VALU 63 %, MFMA 31 %;
// at dk 128 37 % and 30 %; no bank conflict).  bf16, 8 clips x 16 heads, 4096 rows over 2048 keys of which padding leaves about
// three quarters, dk 128: 649 us, 635 TFLOP/s; 4 x 16 heads, 4096 over 4096, dk 64 with a bias: 415 us, 660.  f32, 4 x 8 heads,
// 600 over 1501, padded like that, dk 64: 82 + 6 us in 3 parts, 67 TFLOP/s.  (These and the figures below: medians of one traced run.)
// ---------------------------------------------------------------------------------------------
template <typename T, int DK, bool BIAS>
__global__ void __launch_bounds__(256, DK <= (sizeof(T) == 2 ? 128 : 64) ? 2 : 1) bt_fwd_kernel(BtArgs a) {
  constexpr int KT = tile_rows<T, DK>(), IMG = KT * Img<T, DK>::UPR;
  extern __shared__ uint4 lds[];
  float *mem = (float*)(lds + 4 * IMG), *line = mem + a.distance + LINE_PAD;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t qt = (a.lq + BT_ROWS - 1) / BT_ROWS, items = a.n * a.heads * a.splits * qt, w = work_item(items, a.group * a.splits * qt);
  if (w >= items) return;
  const int row0 = (int)(w % qt) * BT_ROWS + wave * 32, i = row0 + (lane & 31), split = w / qt % a.splits;
  const int ch = w / qt / a.splits, head = ch % a.heads;   // clip heads + head
  const int64_t clip = ch / a.heads;
  const int kt = (a.lk + KT - 1) / KT, per = (kt + a.splits - 1) / a.splits, t0 = split * per, t1 = min(kt, t0 + per);
  const T* kb = (const T*)a.k + clip * a.bk + (int64_t)(head / a.group) * a.hk + (int64_t)t0 * KT * a.ldk;
  const T* vb = (const T*)a.v + clip * a.bv + (int64_t)(head / a.group) * a.hk + (int64_t)t0 * KT * a.ldv;
  const uint8_t* mask = a.mask ? a.mask + clip * a.bmask : nullptr;
  Tile<T, DK, KT> ks, vs;
  ks.start(a.ldk, a.dk);
  vs.start(a.ldv, a.dk);
  uint64_t next = __ballot(t0 < t1 ? mask_byte(mask, t0 * KT, KT, a.lk) : 0);
  if (t0 < t1) {
    ks.load(kb, a.ldk, next, lds);
    vs.load(vb, a.ldv, next, lds + IMG);
  }
  int nb = t0 + 1 < t1 ? mask_byte(mask, (t0 + 1) * KT, KT, a.lk) : 0;
  const bool there = i < a.lq && (!a.q_mask || a.q_mask[clip * a.bq_mask + i]);
  Frag<T, DK> q;
  q.load_rows((const T*)a.q + clip * a.bq + (int64_t)row0 * a.ldq + (int64_t)head * a.hq, a.ldq, a.dk, there);
  if constexpr (BIAS) bias_line(mem, a, head);
  Softmax<DK> sm;
  sm.start();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const uint4 *kimg = lds + buf * 2 * IMG, *vimg = kimg + IMG, *to = lds + (buf ^ 1) * 2 * IMG;
    tile_ready();
    const uint64_t bits = next;
    next = __ballot(nb);
    kb += KT * a.ldk;
    vb += KT * a.ldv;
    if (t + 1 < t1) {   // (no load may be under way when the block ends)
      ks.load(kb, a.ldk, next, to);
      vs.load(vb, a.ldv, next, to + IMG);
    }
    nb = t + 2 < t1 ? mask_byte(mask, (t + 2) * KT, KT, a.lk) : 0;
    if (bits && row0 < a.lq) {
      const int first = t * KT - a.off;
      attend<T, DK, BIAS, KT / 32>(sm, kimg, vimg, q, bits, a, line, first + 4 * h - i, first - (row0 + 31), first + 31 - row0);
    }
  }
  sm.template finish<T>();
  if (a.splits > 1) {   // a part of the keys, laid out for bt_join_kernel
    if (i >= a.lq) return;
    const int tiles = (a.group * a.lq + 31) / 32;
    const int64_t all = (int64_t)a.n * a.kv_heads * tiles * 32;
    const int64_t p = split * all + (clip * a.kv_heads + head / a.group) * tiles * 32 + (int64_t)(head % a.group) * a.lq + i;
    store_row<float, DK>(a.part + p * DK, sm.o, 1.f, DK, true);
    if (h == 0) *(f32x4*)(a.part + a.splits * all * DK + 4 * p) = f32x4{sm.m, sm.l, sm.lr, 0.f};
    return;
  }
  const bool some = there && sm.lr != 0.f;
  const float inv = some ? 1.0f / sm.lr : 0.f;
  if (i >= a.lq) return;
  if (!some)
#pragma unroll
    for (int mb = 0; mb < DK / 32; ++mb) sm.o[mb] = zero16();
  store_row<T, DK>((T*)a.o + clip * a.bo + (int64_t)i * a.ldo + (int64_t)head * a.dk, sm.o, inv, a.dk, a.vec_o);
  if (a.stat) {
    if (h == 0) *(float2*)(a.stat + 2 * ((int64_t)ch * a.lq + i)) = make_float2(some ? sm.m : INFINITY, some ? 1.0f / sm.l : 0.f);
    if (a.o32 != (float*)a.o)
      store_row<float, DK>(a.o32 + ((clip * a.lq + i) * a.heads + head) * a.dk, sm.o, inv, a.dk, a.vec_o);
  }
}

// ---------------------------------------------------------------------------------------------
// forward, few rows: the rows of all heads of a kv head together, 32 a block; the block's waves take every
// fourth tile of 32 keys each, blocks a part of the keys (splits), and the parts are joined by their
// maxima and sums.  Bound by reading the keys and values once: a wave has its next tile in flight
// while it works on one, and needs no barrier for it.  bf16, 8 clips x 32 heads on 8 kv heads, one row over 32773 keys,
// dk 128, three quarters left by padding: 165 + 5 us, 4.9 TB/s; 32 clips x 8 heads over 1200, dk 64, with a bias: 20 + 4 us, 3.9 TB/s.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t few_prow(const BtArgs& a, int64_t pair, int tiles, int tile) { return (pair * tiles + tile) * 32; }

// 4 finished elements of a query row
template <typename T>
__device__ __forceinline__ void few_emit(const BtArgs& a, int64_t clip, int head, int i, int c, f32x4 v) {
  T* row = (T*)a.o + clip * a.bo + (int64_t)i * a.ldo + (int64_t)head * a.dk;
  float* row32 = a.stat && a.o32 != (float*)a.o ? a.o32 + ((clip * a.lq + i) * a.heads + head) * a.dk : nullptr;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < a.dk) {
      row[c + j] = from_f32<T>(v[j]);
      if (row32) row32[c + j] = v[j];
    }
}

template <typename T, int DK, bool BIAS>
__global__ void __launch_bounds__(256, DK <= (sizeof(T) == 2 ? 64 : 32) ? 2 : 1) bt_few_kernel(BtArgs a) {
  constexpr int IMG = 32 * Img<T, DK>::UPR, NU = DK / 4;
  extern __shared__ uint4 lds[];
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = a.group * a.lq, tiles = (rows + 31) / 32, kt = (a.lk + 31) / 32;
  const uint32_t items = a.n * a.kv_heads * a.splits * tiles, w = work_item(items, a.splits * tiles);
  if (w >= items) return;
  const int tile = w % tiles, rest = w / tiles, split = rest % a.splits, pair = rest / a.splits, kvh = pair % a.kv_heads;
  const int64_t clip = pair / a.kv_heads;
  const int r = tile * 32 + (lane & 31), g = min(r, rows - 1) / a.lq, i = min(r, rows - 1) - g * a.lq, head = kvh * a.group + g;
  const bool there = r < rows && (!a.q_mask || a.q_mask[clip * a.bq_mask + i]);
  Frag<T, DK> q;
  q.load((const T*)a.q + clip * a.bq + (int64_t)i * a.ldq + (int64_t)head * a.hq, a.dk, there);
  const int per = (kt + a.splits - 1) / a.splits, end = min(kt, (split + 1) * per);
  int t = split * per + wave;
  const T* kb = (const T*)a.k + clip * a.bk + (int64_t)kvh * a.hk;
  const T* vb = (const T*)a.v + clip * a.bv + (int64_t)kvh * a.hk;
  const uint8_t* mask = a.mask ? a.mask + clip * a.bmask : nullptr;
  uint4 *kimg = lds + wave * 2 * IMG, *vimg = kimg + IMG;
  Softmax<DK> sm;
  sm.start();
  Stage<T, DK, 32, 64> ks, vs;
  auto bytes = [&](int tt) { return tt < end ? mask_byte(mask, tt * 32, 32, a.lk) : 0; };
  uint64_t next = __ballot(bytes(t));
  ks.load(kb + (int64_t)t * 32 * a.ldk, a.ldk, next, a.dk, lane);
  vs.load(vb + (int64_t)t * 32 * a.ldv, a.ldv, next, a.dk, lane);
  int nb = bytes(t + 4);
  for (; t < end; t += 4) {
    ks.store(kimg, lane);
    vs.store(vimg, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the image is the wave's own: its LDS operations run in order
    const uint64_t bits = next;
    next = __ballot(nb);
    ks.load(kb + (int64_t)(t + 4) * 32 * a.ldk, a.ldk, next, a.dk, lane);
    vs.load(vb + (int64_t)(t + 4) * 32 * a.ldv, a.ldv, next, a.dk, lane);
    nb = bytes(t + 8);
    if (bits) {
      f32x16 s = zero16();
      mma_rows<T, DK>(s, kimg, 0, q);
      if constexpr (BIAS) {
        const int rel = t * 32 + 4 * h - (i + a.off), D = a.distance;
        if (__all(rel - 4 * h >= D || rel - 4 * h + 31 <= -D)) {
          const float b = bias_entry(a.table[(int64_t)bucket_of(a, rel > 0 ? 2 * D : 0) * a.heads + head]);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], a.c, b);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int d = min(max(rel + 8 * (e >> 2) + (e & 3), -D), D) + D;
            s[e] = fmaf(s[e], a.c, bias_entry(a.table[(int64_t)bucket_of(a, d) * a.heads + head]));
          }
        }
      }
      if ((uint32_t)bits != 0xFFFFFFFFu) {
        const uint32_t w4 = (uint32_t)bits >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = row_bit(w4, e) ? s[e] : -INFINITY;
      }
      float mt = both_max(max16(s));
      if constexpr (!BIAS) mt *= a.c;
      sm.raise(mt);
      const float m = sm.m == -INFINITY ? 0.f : sm.m;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(BIAS ? s[e] - m : fmaf(s[e], a.c, -m));
        if constexpr (sizeof(T) == 2) sm.l += s[e];
      }
      mma_cols<T, DK, true>(sm.o, vimg, 0, s, &sm.lr);
      if (sizeof(T) == 2) mma_cols<T, DK, true>(sm.o, vimg, 0, unrounded(s), &sm.lr);   // (the few rows' rule is one of BtArgs::fine)
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // join the four waves: o parts as [wave][row][16-byte unit ^ row % 8], maxima and sums behind them
  __syncthreads();
  f32x4* xo = (f32x4*)lds;
  float* xs = (float*)(xo + 4 * 32 * NU);
  sm.template finish<T>();
  if (h == 0) {
    xs[wave * 32 + lane] = sm.m;
    xs[128 + wave * 32 + lane] = sm.l;
    xs[256 + wave * 32 + lane] = sm.lr;
  }
#pragma unroll
  for (int mb = 0; mb < DK / 32; ++mb)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      xo[(wave * 32 + (lane & 31)) * NU + ((8 * mb + 2 * q4 + h) ^ (lane & 7))] =
          f32x4{sm.o[mb][4 * q4], sm.o[mb][4 * q4 + 1], sm.o[mb][4 * q4 + 2], sm.o[mb][4 * q4 + 3]};
  __syncthreads();
  for (int e = tid; e < 32 * NU; e += 256) {
    const int row = e / NU, u = e % NU, rr = tile * 32 + row;
    if (rr >= rows) continue;
    float m = -INFINITY, ls = 0.f, lr = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, xs[k * 32 + row]);
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float mk = xs[k * 32 + row], f = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - m);
      const f32x4 x = xo[(k * 32 + row) * NU + (u ^ (row & 7))];
      const float lk = xs[128 + k * 32 + row];
      ls += lk != lk ? lk : lk * f;   // a part whose scores are NaN has no maximum, and says so by its sum
      lr += lk != lk ? lk : xs[256 + k * 32 + row] * f;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fmaf(x[j], f, v[j]);
    }
    if (a.splits > 1) {
      const int64_t p = (int64_t)split * a.n * a.kv_heads * tiles * 32 + few_prow(a, pair, tiles, tile) + row;
      *(f32x4*)(a.part + p * DK + 4 * u) = v;
      if (u == 0) *(f32x4*)(a.part + (int64_t)a.splits * a.n * a.kv_heads * tiles * 32 * DK + 4 * p) = f32x4{m, ls, lr, 0.f};
      continue;
    }
    const int gg = rr / a.lq, ii = rr - gg * a.lq, hd = kvh * a.group + gg;
    const bool some = lr != 0.f && (!a.q_mask || a.q_mask[clip * a.bq_mask + ii]);
    const float inv = some ? 1.0f / lr : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = some ? v[j] * inv : 0.f;
    few_emit<T>(a, clip, hd, ii, 4 * u, v);
    if (a.stat && u == 0) *(float2*)(a.stat + 2 * ((clip * a.heads + hd) * a.lq + ii)) = make_float2(some ? m : INFINITY, some ? 1.0f / ls : 0.f);
  }
}

// the parts of a row joined: DK / 4 threads a row, the parts in their order
template <typename T, int DK>
__global__ void __launch_bounds__(256) bt_join_kernel(BtArgs a) {
  constexpr int NU = DK / 4;
  const int rows = a.group * a.lq, tiles = (rows + 31) / 32, u = threadIdx.x % NU;
  const int64_t all = (int64_t)a.n * a.kv_heads * tiles * 32, p = (int64_t)blockIdx.x * (256 / NU) + threadIdx.x / NU;
  if (p >= all) return;
  const int64_t pair = p / (tiles * 32), clip = pair / a.kv_heads;
  const int rr = (int)(p % (tiles * 32)), kvh = (int)(pair % a.kv_heads);
  if (rr >= rows) return;
  const float* ml = a.part + (int64_t)a.splits * all * DK;
  float m = -INFINITY, ls = 0.f, lr = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, ml[4 * (s * all + p)]);
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const f32x4 st = *(const f32x4*)(ml + 4 * (s * all + p));
    const float ms = st[0], lk = st[1];
    const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
    const f32x4 x = *(const f32x4*)(a.part + (s * all + p) * DK + 4 * u);
    ls += lk != lk ? lk : lk * f;
    lr += lk != lk ? lk : st[2] * f;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = fmaf(x[j], f, v[j]);
  }
  const int gg = rr / a.lq, ii = rr - gg * a.lq, hd = kvh * a.group + gg;
  const bool some = lr != 0.f && (!a.q_mask || a.q_mask[clip * a.bq_mask + ii]);
  const float inv = some ? 1.0f / lr : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = some ? v[j] * inv : 0.f;
  few_emit<T>(a, clip, hd, ii, 4 * u, v);
  if (a.stat && u == 0) *(float2*)(a.stat + 2 * ((clip * a.heads + hd) * a.lq + ii)) = make_float2(some ? m : INFINITY, some ? 1.0f / ls : 0.f);
}

// ---------------------------------------------------------------------------------------------
// dq (and delta, and the table's gradient): like the forward kernel, a block per 128 query rows of a head.
// Weights stay without their row's 1 / l until the end: it is one factor of the lane's row.
//   Table: ds go into a histogram over clamped distances, a copy a wave (diag_add); blocks past the table's distance
// are summed in registers.
//   Three products a score and one exp: bound by the MFMA and LDS reads that feed it (each 32 keys' image is read twice, by
// rows and transposed).  The forward kernel's sizes: 743 us, 830 TFLOP/s at dk 128 (counters: MFMA 41 %, VALU 38 %); 675 us, 610 at
// dk 64 with the table's gradient (28 %, 53 %); f32 118 + 7 us, 70.
// ---------------------------------------------------------------------------------------------
// the block's histogram copies and its lanes' sums past the distance -> a row of dtab.  first: the block's first query
__device__ __forceinline__ void write_buckets(const BtArgs& a, float* hist, float past, float behind, int first, int64_t row) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, D = a.distance, lines = 2 * D + 1;
  past = group_sum<16>(past);
  behind = group_sum<16>(behind);
  past += __shfl_xor(past, 16);
  behind += __shfl_xor(behind, 16);
  past = both_sum(past);
  behind = both_sum(behind);
  if (lane == 0) {
    hist[wave * lines] = behind;
    hist[wave * lines + 2 * D] = past;
  }
  __syncthreads();
  // the distances that this block's places can have
  const int last = min(a.lq, first + BT_ROWS) - 1;
  const int d0 = max(-D, min(D, -last - a.off)) + D, d1 = max(-D, min(D, a.lk - 1 - first - a.off)) + D;
  int* which = (int*)(hist + lines);   // over the second copy, once it is added to the first
  for (int d = d0 + tid; d <= d1; d += 256) {
    hist[d] = (hist[d] + hist[lines + d]) + (hist[2 * lines + d] + hist[3 * lines + d]);
    which[d] = bucket_of(a, d);
  }
  __syncthreads();
  auto leave = [&](int b, float x) {
    x = group_sum<16>(x);
    x += __shfl_xor(x, 16);
    x = both_sum(x);
    if (lane == 0) a.dtab[row * a.n_buckets + b] = x;
  };
  constexpr int HELD = 8;   // distances a lane holds: most blocks have no more
  if (d1 - d0 < 64 * HELD) {
    float v[HELD];
    int of[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int d = d0 + 64 * k + lane;
      v[k] = d <= d1 ? hist[d] : 0.f;
      of[k] = d <= d1 ? which[d] : -1;
    }
    for (int b = wave; b < a.n_buckets; b += 4) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < HELD; ++k) x += of[k] == b ? v[k] : 0.f;
      leave(b, x);
    }
  } else {
    for (int b = wave; b < a.n_buckets; b += 4) {
      float x = 0.f;
      for (int d = d0 + lane; d <= d1; d += 64) x += which[d] == b ? hist[d] : 0.f;
      leave(b, x);
    }
  }
}

template <typename T, int DK, bool BIAS>
__global__ void __launch_bounds__(256, DK <= (sizeof(T) == 2 ? 128 : 64) ? 2 : 1) bt_dq_kernel(BtArgs a) {
  constexpr int KT = tile_rows<T, DK>(), IMG = KT * Img<T, DK>::UPR, EPU = Img<T, DK>::EPU;
  extern __shared__ uint4 lds[];
  const int lines = 2 * a.distance + 1;
  float *mem = (float*)(lds + 4 * IMG), *line = mem + a.distance + LINE_PAD, *hist = mem + line_floats(a.distance);   // with a table gradient: [4][lines], and the diagonals' images
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t qt = (a.lq + BT_ROWS - 1) / BT_ROWS, items = a.n * a.heads * a.splits * qt, w = work_item(items, a.group * a.splits * qt);
  if (w >= items) return;
  const int first_row = (int)(w % qt) * BT_ROWS, row0 = first_row + wave * 32, i = row0 + (lane & 31), split = w / qt % a.splits;
  const int ch = w / qt / a.splits, head = ch % a.heads, D = a.distance;
  const int64_t clip = ch / a.heads, srow = (int64_t)ch * a.lq + i;   // of the statistics
  const int kt = (a.lk + KT - 1) / KT, per = (kt + a.splits - 1) / a.splits, t0 = split * per, t1 = min(kt, t0 + per);
  const T* kb = (const T*)a.k + clip * a.bk + (int64_t)(head / a.group) * a.hk + (int64_t)t0 * KT * a.ldk;
  const T* vb = (const T*)a.v + clip * a.bv + (int64_t)(head / a.group) * a.hk + (int64_t)t0 * KT * a.ldv;
  const uint8_t* mask = a.mask ? a.mask + clip * a.bmask : nullptr;
  Tile<T, DK, KT> ks, vs;
  ks.start(a.ldk, a.dk);
  vs.start(a.ldv, a.dk);
  uint64_t next = __ballot(t0 < t1 ? mask_byte(mask, t0 * KT, KT, a.lk) : 0);
  if (t0 < t1) {
    ks.load(kb, a.ldk, next, lds);
    vs.load(vb, a.ldv, next, lds + IMG);
  }
  int nb = t0 + 1 < t1 ? mask_byte(mask, (t0 + 1) * KT, KT, a.lk) : 0;
  const bool mine = i < a.lq && (!a.q_mask || a.q_mask[clip * a.bq_mask + i]);
  const float2 st = mine ? *(const float2*)(a.stat + 2 * srow) : make_float2(INFINITY, 0.f);
  const float m = st.x, rl = st.y;
  const bool there = rl != 0.f;   // a row that attends something: of another nothing is read, whatever its do
  Frag<T, DK> q, dO;
  q.load_rows((const T*)a.q + clip * a.bq + (int64_t)row0 * a.ldq + (int64_t)head * a.hq, a.ldq, a.dk, there);
  dO.load_rows((const T*)a.dout + (clip * a.lq + row0) * a.lddo + (int64_t)head * a.hq, a.lddo, a.dk, there);
  const int64_t crow = ((clip * a.lq + i) * a.heads + head) * a.dk;   // of the contiguous rows
  const bool table_grad = BIAS && a.dtable;
  if constexpr (BIAS) {
    bias_line(mem, a, head);
    if (table_grad) {
      for (int d = tid; d < 4 * lines; d += 256) hist[d] = 0.f;
      diag_start(hist + 4 * lines + wave * DIAG);
    }
  }
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < Frag<T, DK>::N; ++s) {
    const uint32_t u[4] = {dO.x[s].x, dO.x[s].y, dO.x[s].z, dO.x[s].w};
#pragma unroll
    for (int f = 0; f < EPU; f += 4) {
      const int c = (2 * s + h) * EPU + f;
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
      if (there) {
        if (a.dk % 4 == 0) {
          if (c < a.dk) o = *(const f32x4*)(a.o32 + crow + c);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < a.dk) o[e] = a.o32[crow + c + e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = sizeof(T) == 4 ? u[e] : e & 1 ? u[(f + e) >> 1] & 0xFFFF0000u : u[(f + e) >> 1] << 16;
        delta = fmaf(__uint_as_float(x), o[e], delta);
      }
    }
  }
  delta = both_sum(delta);
  if (split == 0 && h == 0 && i < a.lq) a.delta[srow] = delta;
  f32x16 acc[DK / 32];
#pragma unroll
  for (int mb = 0; mb < DK / 32; ++mb) acc[mb] = zero16();
  float past = 0.f, behind = 0.f;   // sums of ds at distances >= D, <= -D
  float rest = 0.f, w_past = 0.f;   // (before 1 / l) sums of ds, and of weights at distances >= D
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const uint4 *kimg = lds + buf * 2 * IMG, *vimg = kimg + IMG, *to = lds + (buf ^ 1) * 2 * IMG;
    tile_ready();
    const uint64_t bits = next;
    next = __ballot(nb);
    kb += KT * a.ldk;
    vb += KT * a.ldv;
    if (t + 1 < t1) {
      ks.load(kb, a.ldk, next, to);
      vs.load(vb, a.ldv, next, to + IMG);
    }
    nb = t + 2 < t1 ? mask_byte(mask, (t + 2) * KT, KT, a.lk) : 0;
    if (!bits || row0 >= a.lq) continue;
#pragma unroll
    for (int b = 0; b < KT / 32; ++b) {
      const uint32_t w32 = (uint32_t)(bits >> (32 * b));
      if (!w32) continue;
      f32x16 s = zero16(), dp = zero16();
      mma_rows<T, DK>(s, kimg, 32 * b, q);
      mma_rows<T, DK>(dp, vimg, 32 * b, dO);
      const int first = t * KT + 32 * b - a.off, lo = first - (row0 + 31), hi = first + 31 - row0;
      float f = a.c, e = -m;   // scores less the maximum, in log2 units: f s + e
      if constexpr (BIAS) {
        float bias = 0.f;
        if (!one_bias(line, D, lo, hi, bias)) {
          add_bias<1>(s, line, a.c, first + 4 * h - i, D, lo, hi);
          f = 1.f;
        }
        e += bias;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], f, e));
      if (w32 != 0xFFFFFFFFu) {
        const uint32_t w4 = w32 >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = row_bit(w4, r) ? s[r] : 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = s[r] * (dp[r] - delta);
      if constexpr (BIAS) {
        if (table_grad) {
          if (past_table(D, lo, hi)) {
            float x = 0.f, y = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) x += dp[r];
            rest += x;
            if (lo >= D) {
              past = fmaf(x, rl, past);
#pragma unroll
              for (int r = 0; r < 16; ++r) y += s[r];
              w_past += y;
            } else {
              behind = fmaf(x, rl, behind);
            }
          } else {
            f32x16 x;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              rest += dp[r];
              x[r] = dp[r] * rl;
            }
            if (hi >= D)
#pragma unroll
              for (int r = 0; r < 16; ++r) w_past += first + reg_row(r, h) - i >= D ? s[r] : 0.f;
            diag_add(hist + 4 * lines + wave * DIAG, hist + wave * lines + D, x, first - row0, D, past, behind);
          }
        }
      }
      mma_cols<T, DK>(acc, kimg, 32 * b, dp);
      if (sizeof(T) == 2 && a.fine) mma_cols<T, DK>(acc, kimg, 32 * b, unrounded(dp));
    }
  }
  if (i < a.lq) {
    if (!there)
#pragma unroll
      for (int mb = 0; mb < DK / 32; ++mb) acc[mb] = zero16();
    if (a.splits == 1) store_row<T, DK>((T*)a.dq + crow, acc, a.scale * rl, a.dk, a.vec_o);
    else store_row<float, DK>(a.part + (int64_t)split * a.n * a.lq * a.heads * a.dk + crow, acc, a.scale * rl, a.dk, a.vec_o);
  }
  if constexpr (BIAS) {
    if (table_grad) {
      if constexpr (sizeof(T) == 2) {
        rest = both_sum(rest) * rl;
        w_past = both_sum(w_past) * rl;
        if (h == 0 && i < a.lq) {
          const int64_t all = (int64_t)a.n * a.heads * a.lq;
          a.rest[2 * split * all + srow] = rest;
          a.rest[(2 * split + 1) * all + srow] = w_past;
        }
      }
      __syncthreads();   // (a part without a tile has passed no barrier since the copies were cleared)
      write_buckets(a, hist, past, behind, first_row, w);
    }
  }
}

// The rest of a bf16 table gradient.  delta comes from an o whose weights were rounded, and an error e_i of delta is
// common to its row's ds: the dq and dk sums round each ds to bf16 and do not see it, but the table's gradient is an
// f32 sum of many.  ds sum to zero over a row, so that what they do sum to is e_i, and each ds has p_ij e_i too
// much: this kernel takes sum_i p_ij e_i off each distance's sum.  Only the places within the table's distance
// are formed again (scores alone); the weights past it were summed on the way, and those behind are the remainder to 1.
// 80 us of 4 x 16 heads, 4096 x 4096, distance 128, whose dq takes 675; 36 beside 58 at 6 x 12 heads, 777 x 777, distance 200.
template <typename T, int DK>
__global__ void __launch_bounds__(256, 2) bt_table_rest_kernel(BtArgs a) {
  constexpr int KT = tile_rows<T, DK>(), IMG = KT * Img<T, DK>::UPR;
  extern __shared__ uint4 lds[];
  const int lines = 2 * a.distance + 1, D = a.distance;
  float *mem = (float*)(lds + 2 * IMG), *line = mem + D + LINE_PAD, *hist = mem + line_floats(D);
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t qt = (a.lq + BT_ROWS - 1) / BT_ROWS, items = a.n * a.heads * qt, w = work_item(items, a.group * qt);
  if (w >= items) return;
  const int first = (int)(w % qt) * BT_ROWS, row0 = first + wave * 32, i = row0 + (lane & 31), ch = w / qt, head = ch % a.heads;
  const int64_t clip = ch / a.heads, all = (int64_t)a.n * a.heads * a.lq, srow = (int64_t)ch * a.lq + i;
  // keys within the distance of one of the block's queries: j - i - off in -D + 1 .. D - 1
  const int64_t j0 = (int64_t)first + a.off - D + 1, j1 = (int64_t)min(first + BT_ROWS, a.lq) - 1 + a.off + D;
  const int t0 = (int)max((int64_t)0, min(j0, (int64_t)a.lk)) / KT, t1 = (int)((max((int64_t)0, min(j1, (int64_t)a.lk)) + KT - 1) / KT);
  const T* kb = (const T*)a.k + clip * a.bk + (int64_t)(head / a.group) * a.hk + (int64_t)t0 * KT * a.ldk;
  const uint8_t* mask = a.mask ? a.mask + clip * a.bmask : nullptr;
  Tile<T, DK, KT> ks;
  ks.start(a.ldk, a.dk);
  uint64_t next = __ballot(t0 < t1 ? mask_byte(mask, t0 * KT, KT, a.lk) : 0);
  if (t0 < t1) ks.load(kb, a.ldk, next, lds);
  int nb = t0 + 1 < t1 ? mask_byte(mask, (t0 + 1) * KT, KT, a.lk) : 0;
  const bool mine = i < a.lq && (!a.q_mask || a.q_mask[clip * a.bq_mask + i]);
  const float2 st = mine ? *(const float2*)(a.stat + 2 * srow) : make_float2(INFINITY, 0.f);
  const float m = st.x, rl = st.y;
  Frag<T, DK> q;
  q.load_rows((const T*)a.q + clip * a.bq + (int64_t)row0 * a.ldq + (int64_t)head * a.hq, a.ldq, a.dk, mine);
  float e = 0.f, past = 0.f, near = 0.f;   // near: weights before 1 / l
  if (mine)
    for (int s = 0; s < a.splits; ++s) {
      e += a.rest[2 * s * all + srow];
      past += a.rest[(2 * s + 1) * all + srow];
    }
  const float back = -e * rl;   // (a row that attends nothing: 0, and its maximum is infinite)
  bias_line(mem, a, head);
  for (int d = tid; d < 4 * lines; d += 256) hist[d] = 0.f;
  diag_start(hist + 4 * lines + wave * DIAG);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const uint4* kimg = lds + buf * IMG;
    tile_ready();
    const uint64_t bits = next;
    next = __ballot(nb);
    kb += KT * a.ldk;
    if (t + 1 < t1) ks.load(kb, a.ldk, next, lds + (buf ^ 1) * IMG);
    nb = t + 2 < t1 ? mask_byte(mask, (t + 2) * KT, KT, a.lk) : 0;
    if (!bits || row0 >= a.lq) continue;
#pragma unroll
    for (int b = 0; b < KT / 32; ++b) {
      const uint32_t w32 = (uint32_t)(bits >> (32 * b));
      const int at = t * KT + 32 * b - a.off, rel = at + 4 * h - i, lo = at - (row0 + 31), hi = at + 31 - row0;
      if (!w32 || past_table(D, lo, hi)) continue;
      f32x16 s = zero16();
      mma_rows<T, DK>(s, kimg, 32 * b, q);
      add_bias<1>(s, line, a.c, rel, D, lo, hi);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - m);
      if (w32 != 0xFFFFFFFFu) {
        const uint32_t w4 = w32 >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = row_bit(w4, r) ? s[r] : 0.f;
      }
      if (lo <= -D || hi >= D) {   // places past the distance are not this kernel's
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = rel + 8 * (r >> 2) + (r & 3);
          s[r] = d < D && d > -D ? s[r] : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        near += s[r];
        s[r] *= back;
      }
      float none = 0.f;
      diag_add(hist + 4 * lines + wave * DIAG, hist + wave * lines + D, s, at - row0, D, none, none);
    }
  }
  near = both_sum(near) * rl;
  const bool counts = h == 0 && rl != 0.f;
  const float behind = counts ? -e * (1.f - past - near) : 0.f;
  past = counts ? -e * past : 0.f;
  __syncthreads();
  write_buckets(a, hist, past, behind, first, items * a.splits + w);
}

// the blocks' table gradients: a wave per head and bucket, lanes over the blocks, then a fixed tree.  per: blocks of a clip
// and head in the first list, per2 in the second behind it
static __global__ void __launch_bounds__(64) bt_table_kernel(BtArgs a, int per, int per2) {
  const int head = blockIdx.x % a.heads, b = blockIdx.x / a.heads, lane = threadIdx.x;
  double x = 0.;
  for (int64_t e = lane; e < (int64_t)a.n * per; e += 64)
    x += a.dtab[((e / per * a.heads + head) * per + e % per) * a.n_buckets + b];
  const float* second = a.dtab + (int64_t)a.n * a.heads * per * a.n_buckets;
  for (int64_t e = lane; e < (int64_t)a.n * per2; e += 64)
    x += second[((e / per2 * a.heads + head) * per2 + e % per2) * a.n_buckets + b];
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if (lane == 0) a.dtable[b * a.heads + head] = (float)x;
}

// ---------------------------------------------------------------------------------------------
// dk, dv: a block per 128 keys of a kv head; the queries of all its heads are streamed, head after head, so that
// a shared head's gradient is one sum in registers.  Four products a score.  bf16 at dk 64 runs two waves a SIMD (4 x 16 heads,
// 4096 x 4096: 717 us, 765 TFLOP/s; counters: MFMA 36 %, VALU 48 %); past 64 it has a kernel of its own below.  f32, 4 x 8 heads, 600 x 1501, dk 64: 167 us, 66 TFLOP/s.
// ---------------------------------------------------------------------------------------------
template <typename T, int DK, bool BIAS>
__global__ void __launch_bounds__(256, DK <= (sizeof(T) == 2 ? 64 : 32) ? 2 : 1) bt_dkv_kernel(BtArgs a) {
  constexpr int QT = tile_rows<T, DK>(), IMG = QT * Img<T, DK>::UPR;
  extern __shared__ uint4 lds[];
  // [2][q, do images], [2][3][QT] statistics (maximum, 1 / sum, delta), the bias line
  float *stats = (float*)(lds + 4 * IMG), *mem = stats + 6 * QT, *line = mem + a.distance + LINE_PAD;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tiles = (a.lk + BT_ROWS - 1) / BT_ROWS, items = a.n * a.kv_heads * a.splits * tiles, w = work_item(items, a.splits * tiles);
  if (w >= items) return;
  const int key0 = (int)(w % tiles) * BT_ROWS, row0 = key0 + wave * 32, j = row0 + (lane & 31), split = w / tiles % a.splits;
  const int pair = w / tiles / a.splits, kvh = pair % a.kv_heads, D = a.distance;
  const int64_t clip = pair / a.kv_heads;
  const uint8_t* mask = a.mask ? a.mask + clip * a.bmask : nullptr;
  const bool any = __ballot(mask_byte(mask, key0, 64, a.lk)) | __ballot(mask_byte(mask, key0 + 64, 64, a.lk));
  const bool there = j < a.lk && (!mask || mask[j]);
  const bool live = __ballot(there);
  Frag<T, DK> k, v;
  k.load_rows((const T*)a.k + clip * a.bk + (int64_t)row0 * a.ldk + (int64_t)kvh * a.hk, a.ldk, a.dk, there);
  v.load_rows((const T*)a.v + clip * a.bv + (int64_t)row0 * a.ldv + (int64_t)kvh * a.hk, a.ldv, a.dk, there);
  f32x16 dk[DK / 32], dv[DK / 32];
#pragma unroll
  for (int mb = 0; mb < DK / 32; ++mb) dk[mb] = dv[mb] = zero16();
  const int qt = (a.lq + QT - 1) / QT, steps = a.group * qt, per = (steps + a.splits - 1) / a.splits;
  const int s0 = any ? split * per : 0, s1 = any ? min(steps, s0 + per) : 0;
  const uint8_t* q_mask = a.q_mask ? a.q_mask + clip * a.bq_mask : nullptr;
  Tile<T, DK, QT> qs, os;
  qs.start(a.ldq, a.dk);
  os.start(a.lddo, a.dk);
  float st_m = 0.f, st_r = 0.f, st_d = 0.f;
  auto load = [&](int step, uint64_t bits, const uint4* img) {
    const int head = kvh * a.group + step / qt, i0 = step % qt * QT;
    qs.load((const T*)a.q + clip * a.bq + (int64_t)i0 * a.ldq + (int64_t)head * a.hq, a.ldq, bits, img);
    os.load((const T*)a.dout + (clip * a.lq + i0) * a.lddo + (int64_t)head * a.hq, a.lddo, bits, img + IMG);
    if (tid < QT) {
      const int64_t at = (clip * a.heads + head) * a.lq + i0 + tid;
      const bool row = (bits >> tid) & 1;
      st_m = row ? a.stat[2 * at] : INFINITY;
      st_r = row ? a.stat[2 * at + 1] : 0.f;
      st_d = row ? a.delta[at] : 0.f;
    }
  };
  auto put = [&](float* sts) {
    if (tid < QT) {
      sts[tid] = st_m;
      sts[QT + tid] = st_r;
      sts[2 * QT + tid] = st_d;
    }
  };
  auto bytes = [&](int step) { return step < s1 ? mask_byte(q_mask, step % qt * QT, QT, a.lq) : 0; };
  uint64_t next = __ballot(bytes(s0));
  if (s0 < s1) {
    load(s0, next, lds);
    put(stats);
  }
  int nb = bytes(s0 + 1), lined = -1;
  for (int t = s0; t < s1; ++t) {
    const int buf = (t - s0) & 1;
    const uint4 *qimg = lds + buf * 2 * IMG, *oimg = qimg + IMG;
    const float* sts = stats + buf * 3 * QT;
    if constexpr (BIAS) {
      if (t / qt != lined) {   // another head: its line, once all have done with the last one's
        __syncthreads();
        lined = t / qt;
        bias_line(mem, a, kvh * a.group + lined);
      }
    }
    tile_ready();
    const uint64_t bits = next;
    next = __ballot(nb);
    if (t + 1 < s1) load(t + 1, next, lds + (buf ^ 1) * 2 * IMG);
    nb = bytes(t + 2);
    if (bits && live) {
#pragma unroll
    for (int b = 0; b < QT / 32; ++b) {
      if (!(uint32_t)(bits >> (32 * b))) continue;
      f32x16 s = zero16(), dp = zero16();
      mma_rows<T, DK>(s, qimg, 32 * b, k);
      mma_rows<T, DK>(dp, oimg, 32 * b, v);
      if constexpr (BIAS) {
        const int q0 = t % qt * QT + 32 * b + a.off;   // position of the block's first query
        add_bias<-1>(s, line, a.c, j - (q0 + 4 * h), D, row0 - (q0 + 31), row0 + 31 - q0);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * b + 8 * g + 4 * h;
        const f32x4 m = *(const f32x4*)(sts + at), rl = *(const f32x4*)(sts + QT + at), dl = *(const f32x4*)(sts + 2 * QT + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          s[r] = __builtin_amdgcn_exp2f(BIAS ? s[r] - m[e] : fmaf(s[r], a.c, -m[e])) * rl[e];
          dp[r] = s[r] * (dp[r] - dl[e]);
        }
      }
      mma_cols<T, DK>(dv, oimg, 32 * b, s);
      mma_cols<T, DK>(dk, qimg, 32 * b, dp);
      if (sizeof(T) == 2 && a.fine) {
        mma_cols<T, DK>(dv, oimg, 32 * b, unrounded(s));
        mma_cols<T, DK>(dk, qimg, 32 * b, unrounded(dp));
      }
    }
    }
    put(stats + (buf ^ 1) * 3 * QT);
  }
  if (j >= a.lk) return;
  if (!there)
#pragma unroll
    for (int mb = 0; mb < DK / 32; ++mb) dk[mb] = dv[mb] = zero16();
  const int64_t row = ((clip * a.lk + j) * a.kv_heads + kvh) * a.dk, all = (int64_t)a.n * a.lk * a.kv_heads * a.dk;
  if (a.splits == 1) {
    store_row<T, DK>((T*)a.dk_out + row, dk, a.scale, a.dk, a.vec_o);
    store_row<T, DK>((T*)a.dv + row, dv, 1.f, a.dk, a.vec_o);
  } else {
    store_row<float, DK>(a.part + split * all + row, dk, a.scale, a.dk, a.vec_o);
    store_row<float, DK>(a.part + (a.splits + split) * all + row, dv, 1.f, a.dk, a.vec_o);
  }
}

// ---------------------------------------------------------------------------------------------
// dk, dv of bf16 heads past 64: two sums and two stationary rows are 400 registers, and one wave a SIMD overlaps nothing with its
// products (1350 us at 8 clips x 4 kv heads of 4, 4096 x 2048, dk 128, padded; 1206 with this kernel in the same run).  So two waves share 32 keys: the first holds k and dv,
// forms the weights, p^T do and hands the weights on in f32 through LDS; the second, 32 queries behind, holds v and dk, forms
// dp, ds and ds^T q.  Each has two of the four products, and a SIMD two waves.  A tile is in use for one and a half rounds: three
// buffers.  Traced 1243 us, 660 TFLOP/s (counters: MFMA 31 %, VALU 27 %); what is left are the barrier after each 32 queries and the VALU
// work beside the products.
// ---------------------------------------------------------------------------------------------
template <bool BIAS>
__global__ void __launch_bounds__(512, 2) bt_dkv_pair_kernel(BtArgs a) {
  typedef bf16_t T;
  constexpr int DK = 128, QT = tile_rows<T, DK>(), IMG = QT * Img<T, DK>::UPR;
  static_assert(QT == 64, "two blocks of 32 queries a tile");
  extern __shared__ uint4 lds[];
  // [3][q, do images], [4 pairs][2 blocks][4][64 lanes] weights, [3][3][QT] statistics (maximum, 1 / sum, delta), the bias line
  f32x4* weights = (f32x4*)(lds + 6 * IMG);
  float *stats = (float*)(weights + 4 * 2 * 4 * 64), *mem = stats + 9 * QT, *line = mem + a.distance + LINE_PAD;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tiles = (a.lk + BT_ROWS - 1) / BT_ROWS, items = a.n * a.kv_heads * a.splits * tiles, w = work_item(items, a.splits * tiles);
  if (w >= items) return;
  const int key0 = (int)(w % tiles) * BT_ROWS, row0 = key0 + (wave & 3) * 32, j = row0 + (lane & 31), split = w / tiles % a.splits;
  const int pair = w / tiles / a.splits, kvh = pair % a.kv_heads, D = a.distance;
  const int64_t clip = pair / a.kv_heads;
  const uint8_t* mask = a.mask ? a.mask + clip * a.bmask : nullptr;
  const bool any = __ballot(mask_byte(mask, key0, 64, a.lk)) | __ballot(mask_byte(mask, key0 + 64, 64, a.lk));
  const bool there = j < a.lk && (!mask || mask[j]);
  const bool live = __ballot(there);
  auto work = [&](auto which) {   // (the two ways apart, so that each has its registers to itself)
    constexpr bool second = decltype(which)::value;
    Frag<T, DK> own;   // k, v
    const int64_t ld = second ? a.ldv : a.ldk;
    own.load_rows((second ? (const T*)a.v + clip * a.bv : (const T*)a.k + clip * a.bk) + (int64_t)row0 * ld + (int64_t)kvh * a.hk, ld, a.dk, there);
    f32x16 acc[DK / 32];   // dv, dk
#pragma unroll
    for (int mb = 0; mb < DK / 32; ++mb) acc[mb] = zero16();
    const int qt = (a.lq + QT - 1) / QT, steps = a.group * qt, per = (steps + a.splits - 1) / a.splits;
    const int s0 = any ? split * per : 0, s1 = any ? min(steps, s0 + per) : 0;
    const uint8_t* q_mask = a.q_mask ? a.q_mask + clip * a.bq_mask : nullptr;
    Tile<T, DK, QT> rows;   // the first waves load q, the second do
    const int64_t ldr = second ? a.lddo : a.ldq;
    rows.start(ldr, a.dk);
    float st_m = 0.f, st_r = 0.f, st_d = 0.f;
    auto load = [&](int step, uint64_t bits, int buf) {
      const int head = kvh * a.group + step / qt, i0 = step % qt * QT;
      const T* from = second ? (const T*)a.dout + clip * a.lq * a.lddo : (const T*)a.q + clip * a.bq;
      rows.load(from + (int64_t)i0 * ldr + (int64_t)head * a.hq, ldr, bits, lds + (2 * buf + second) * IMG);
      if (!second && tid < QT) {
        const int64_t at = (clip * a.heads + head) * a.lq + i0 + tid;
        const bool row = (bits >> tid) & 1;
        st_m = row ? a.stat[2 * at] : INFINITY;
        st_r = row ? a.stat[2 * at + 1] : 0.f;
        st_d = row ? a.delta[at] : 0.f;
      }
    };
    auto put = [&](int buf) {
      float* sts = stats + buf * 3 * QT;
      if (!second && tid < QT) {
        sts[tid] = st_m;
        sts[QT + tid] = st_r;
        sts[2 * QT + tid] = st_d;
      }
    };
    auto bytes = [&](int step) { return step < s1 ? mask_byte(q_mask, step % qt * QT, QT, a.lq) : 0; };
    // queries 32 b .. of tile t, whose bits are bits: the first wave's half, and the second's
    auto first_half = [&](int t, int buf, int b, uint64_t bits) {
      if (!(uint32_t)(bits >> (32 * b))) return;
      const uint4 *qimg = lds + buf * 2 * IMG, *oimg = qimg + IMG;
      const float* sts = stats + buf * 3 * QT;
      f32x16 s = zero16();
      mma_rows<T, DK>(s, qimg, 32 * b, own);
      if constexpr (BIAS) {
        const int q0 = t % qt * QT + 32 * b + a.off;   // position of the block's first query
        add_bias<-1>(s, line, a.c, j - (q0 + 4 * h), D, row0 - (q0 + 31), row0 + 31 - q0);
      }
      f32x4* out = weights + ((wave & 3) * 2 + b) * 4 * 64 + lane;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * b + 8 * g + 4 * h;
        const f32x4 m = *(const f32x4*)(sts + at), rl = *(const f32x4*)(sts + QT + at);
        f32x4 p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          p[e] = s[r] = __builtin_amdgcn_exp2f(BIAS ? s[r] - m[e] : fmaf(s[r], a.c, -m[e])) * rl[e];
        }
        out[64 * g] = p;
      }
      mma_cols<T, DK>(acc, oimg, 32 * b, s);
      if (a.fine) mma_cols<T, DK>(acc, oimg, 32 * b, unrounded(s));
    };
    auto second_half = [&](int buf, int b, uint64_t bits) {
      if (!(uint32_t)(bits >> (32 * b))) return;
      const uint4 *qimg = lds + buf * 2 * IMG, *oimg = qimg + IMG;
      const float* sts = stats + buf * 3 * QT + 2 * QT;
      f32x16 dp = zero16();
      mma_rows<T, DK>(dp, oimg, 32 * b, own);
      const f32x4* in = weights + ((wave & 3) * 2 + b) * 4 * 64 + lane;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 p = in[64 * g], dl = *(const f32x4*)(sts + 32 * b + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[4 * g + e] = p[e] * (dp[4 * g + e] - dl[e]);
      }
      mma_cols<T, DK>(acc, qimg, 32 * b, dp);
      if (a.fine) mma_cols<T, DK>(acc, qimg, 32 * b, unrounded(dp));
    };
    uint64_t next = __ballot(bytes(s0)), before = 0;   // bits of the next tile and of the last
    if (s0 < s1) {
      load(s0, next, 0);
      put(0);
    }
    int nb = bytes(s0 + 1), lined = -1, buf = 0, last = 0;
    for (int t = s0; t < s1; ++t) {
      const int to = buf == 2 ? 0 : buf + 1;
      if constexpr (BIAS) {
        if (t / qt != lined) {   // another head: its line, once all have done with the last one's
          lds_ready();
          lined = t / qt;
          bias_line(mem, a, kvh * a.group + lined);
        }
      }
      tile_ready();
      const uint64_t bits = next;
      next = __ballot(nb);
      if (t + 1 < s1) load(t + 1, next, to);
      nb = bytes(t + 2);
      if (live) {
        if constexpr (second) second_half(last, 1, before);
        else first_half(t, buf, 0, bits);
      }
      lds_ready();
      if (live) {
        if constexpr (second) second_half(buf, 0, bits);
        else first_half(t, buf, 1, bits);
      }
      put(to);
      before = bits;
      last = buf;
      buf = to;
    }
    lds_ready();
    if constexpr (second)
      if (live) second_half(last, 1, before);
    if (j >= a.lk) return;
    if (!there)
#pragma unroll
      for (int mb = 0; mb < DK / 32; ++mb) acc[mb] = zero16();
    const int64_t row = ((clip * a.lk + j) * a.kv_heads + kvh) * a.dk, all = (int64_t)a.n * a.lk * a.kv_heads * a.dk;
    const float scale = second ? a.scale : 1.f;
    if (a.splits == 1) store_row<T, DK>((T*)(second ? a.dk_out : a.dv) + row, acc, scale, a.dk, a.vec_o);
    else store_row<float, DK>(a.part + (second ? split : a.splits + split) * all + row, acc, scale, a.dk, a.vec_o);
  };
  if (wave < 4) work(std::false_type{});
  else work(std::true_type{});
}

// rows of heads that are not whole aligned 16-byte units, laid out anew as such: (clips rows heads) dkp elements, zeros past dk
template <typename T>
__global__ void __launch_bounds__(256) bt_pack_kernel(int64_t n, int rows, int heads, int dk, int dkp, const T* __restrict__ src, int64_t ld,
                                                      int64_t b, T* __restrict__ dst) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int c = (int)(e % dkp);
    const int64_t r = e / dkp / heads;
    dst[e] = c < dk ? src[r / rows * b + r % rows * ld + (e / dkp % heads) * dk + c] : (T)0;
  }
}

// out = the sum of the splits' parts, in their order
template <typename T>
__global__ void __launch_bounds__(256) bt_sum_kernel(int64_t n, int splits, const float* __restrict__ part, T* __restrict__ out) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    float x = 0.f;
    for (int s = 0; s < splits; ++s) x += part[s * n + e];
    out[e] = from_f32<T>(x);
  }
}

// ---------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------
template <typename T>
hipError_t sum_parts(int64_t n, int splits, const float* part, void* out, hipStream_t s) {
  hipLaunchKernelGGL(bt_sum_kernel<T>, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096)), dim3(256), 0, s, n, splits, part, (T*)out);
  return hipGetLastError();
}

template <typename T>
hipError_t pack_rows(const BtArgs& a, const void* src, int64_t ld, int64_t b, int rows, int heads, void* dst, hipStream_t s) {
  constexpr int per = 16 / sizeof(T);
  const int dkp = (a.dk + per - 1) / per * per;
  const int64_t n = (int64_t)a.n * rows * heads * dkp;
  hipLaunchKernelGGL(bt_pack_kernel<T>, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 8192)), dim3(256), 0, s, n, rows, heads, a.dk, dkp,
                     (const T*)src, ld, b, (T*)dst);
  return hipGetLastError();
}

template <typename T, int DK, bool BIAS>
struct Kernels {
  static constexpr int KT = tile_rows<T, DK>();
  static constexpr size_t IMAGES = 4 * (size_t)KT * Img<T, DK>::UPR * 16;
  static size_t lines(const BtArgs& a) { return BIAS ? line_floats(a.distance) * sizeof(float) : 0; }

  static size_t table_lds(const BtArgs& a) { return lines(a) + (4 * (2 * (size_t)a.distance + 1) + 4 * DIAG) * sizeof(float); }

  static void join(const BtArgs& a, hipStream_t s) {
    const uint32_t rows = (a.group * a.lq + 31) / 32 * 32 * a.n * a.kv_heads;
    hipLaunchKernelGGL((bt_join_kernel<T, DK>), dim3((rows + 1024 / DK - 1) / (1024 / DK)), dim3(256), 0, s, a);
  }
  static hipError_t fwd(const BtArgs& a, hipStream_t s) {
    static std::atomic<bool> done[64];
    const size_t lds = IMAGES + lines(a);
    if (const hipError_t e = allow_lds(bt_fwd_kernel<T, DK, BIAS>, lds, done)) return e;
    const uint32_t each = a.group * ((a.lq + BT_ROWS - 1) / BT_ROWS) * a.splits;
    hipLaunchKernelGGL((bt_fwd_kernel<T, DK, BIAS>), dim3(work_grid(a.n * a.kv_heads * each, each)), dim3(256), lds, s, a);
    if (a.splits > 1) join(a, s);
    return hipGetLastError();
  }
  static hipError_t few(const BtArgs& a, hipStream_t s) {
    static std::atomic<bool> done[64];
    // the four waves' images, which then hold the four parts of o (f32) and 384 statistics
    const size_t lds = std::max<size_t>(4 * 2 * 32 * Img<T, DK>::UPR * 16, 4 * 32 * DK * sizeof(float)) + 1536;
    if (const hipError_t e = allow_lds(bt_few_kernel<T, DK, BIAS>, lds, done)) return e;
    const uint32_t tiles = (a.group * a.lq + 31) / 32, rows = tiles * a.n * a.kv_heads;
    hipLaunchKernelGGL((bt_few_kernel<T, DK, BIAS>), dim3(work_grid(rows * a.splits, a.splits * tiles)), dim3(256), lds, s, a);
    if (a.splits > 1) join(a, s);
    return hipGetLastError();
  }
  static hipError_t dq(const BtArgs& a, hipStream_t s) {
    static std::atomic<bool> done[64];
    const size_t lds = IMAGES + (a.dtable ? table_lds(a) : lines(a));
    if (const hipError_t e = allow_lds(bt_dq_kernel<T, DK, BIAS>, lds, done)) return e;
    const uint32_t qt = (a.lq + BT_ROWS - 1) / BT_ROWS, each = a.group * qt;
    hipLaunchKernelGGL((bt_dq_kernel<T, DK, BIAS>), dim3(work_grid(a.n * a.kv_heads * each * a.splits, each * a.splits)), dim3(256), lds, s, a);
    if (const hipError_t e = hipGetLastError()) return e;
    if constexpr (BIAS) {
      if (a.dtable) {
        if constexpr (sizeof(T) == 2) {
          static std::atomic<bool> rest_done[64];
          const size_t rest_lds = IMAGES / 2 + table_lds(a);
          if (const hipError_t e = allow_lds(bt_table_rest_kernel<T, DK>, rest_lds, rest_done)) return e;
          hipLaunchKernelGGL((bt_table_rest_kernel<T, DK>), dim3(work_grid(a.n * a.kv_heads * each, each)), dim3(256), rest_lds, s, a);
        }
        hipLaunchKernelGGL(bt_table_kernel, dim3(a.heads * a.n_buckets), dim3(64), 0, s, a, (int)(qt * a.splits), sizeof(T) == 2 ? (int)qt : 0);
        if (const hipError_t e = hipGetLastError()) return e;
      }
    }
    return a.splits > 1 ? sum_parts<T>((int64_t)a.n * a.lq * a.heads * a.dk, a.splits, a.part, a.dq, s) : hipSuccess;
  }
  static hipError_t dkv(const BtArgs& a, hipStream_t s) {
    static std::atomic<bool> done[64];
    const uint32_t each = (a.lk + BT_ROWS - 1) / BT_ROWS * a.splits, grid = work_grid(a.n * a.kv_heads * each, each);
    if constexpr (sizeof(T) == 2 && DK == 128) {
      const size_t lds = IMAGES / 2 * 3 + 4 * 2 * 4 * 64 * sizeof(f32x4) + 9 * KT * sizeof(float) + lines(a);
      if (const hipError_t e = allow_lds(bt_dkv_pair_kernel<BIAS>, lds, done)) return e;
      hipLaunchKernelGGL((bt_dkv_pair_kernel<BIAS>), dim3(grid), dim3(512), lds, s, a);
    } else {
      const size_t lds = IMAGES + 6 * KT * sizeof(float) + lines(a);
      if (const hipError_t e = allow_lds(bt_dkv_kernel<T, DK, BIAS>, lds, done)) return e;
      hipLaunchKernelGGL((bt_dkv_kernel<T, DK, BIAS>), dim3(grid), dim3(256), lds, s, a);
    }
    if (const hipError_t e = hipGetLastError()) return e;
    if (a.splits == 1) return hipSuccess;
    const int64_t all = (int64_t)a.n * a.lk * a.kv_heads * a.dk;
    if (const hipError_t e = sum_parts<T>(all, a.splits, a.part, a.dk_out, s)) return e;
    return sum_parts<T>(all, a.splits, a.part + a.splits * all, a.dv, s);
  }
  static constexpr Launch launch = {pack_rows<T>, fwd, few, dq, dkv};
};

template <typename T>
const Launch& pick(const BtArgs& a) {
  if (a.table) return a.dk <= 32 ? Kernels<T, 32, true>::launch : a.dk <= 64 ? Kernels<T, 64, true>::launch : Kernels<T, 128, true>::launch;
  return a.dk <= 32 ? Kernels<T, 32, false>::launch : a.dk <= 64 ? Kernels<T, 64, false>::launch : Kernels<T, 128, false>::launch;
}

}  // namespace battn
}  // namespace ggd
