// ggd_resnorm.hip -- the norms around a decoder block fused with its gate and residual scale (gfx950):
//   h' = scale h + gate * post(y),  u = pre(h')     (include/ggd_train.h, ggd_tr_resnorm_fwd / _bwd)
// post / pre: LayerNorm or RMS norm with f32 weights; gate: none, one row for all, one per group of
// rows (a clip) or one per row.
//
// Every quantity of a row is a function of that row alone but for the weights' and the gate's
// gradients, so both passes are one read of each row tensor and one write of each result: bound by
// HBM.  A row lives in registers between its reductions -- a wave's (d <= 1024) or a block's -- and
// the statistics are two-pass (mean, then the centred squares) on those registers in f32.
#include "ggd_common.h"

#include <algorithm>
#include <cstdint>

#include "../../include/ggd_train.h"

namespace ggd {
namespace {

constexpr int RN_MAX_D = 8192;
constexpr int64_t RN_MAX_GRID = 1 << 22;   // blocks of a launch; its threads fit 32 bits
constexpr int64_t RN_MAX_ROWS = INT32_MAX;   // a row's number fits 32 bits, an element's offset need not

struct RnFwd {
  int64_t rows, gate_rows;
  int d, rms;
  float scale, eps;
  const void *h, *y, *gate;
  const float *pg, *pb, *ng, *nb;  // post weights (pg null: no post norm), pre weights
  void *ho, *u;
  float* stats;  // [4][rows]: post mean, post 1 / sd, pre mean, pre 1 / sd (null: not kept)
};

struct RnBwd {
  RnFwd f;
  const void *dho, *du;
  void *dh, *dy, *dgate;
  float* part;  // [5][blocks][d]: pre weight, pre bias, post weight, post bias, gate sums of each block
  int64_t seg, segs;   // rows of a block, all of one gate row, and blocks of a gate row
  int64_t per, groups; // per > 0: a block has `per` whole gate rows of the `groups` there are instead, and writes their sums itself
  int64_t group_rows;  // rows of a gate row (all rows without a gate, and where each row has its own)
  bool by_row;         // each row has its own gate row
};

// the thread's elements of a row: vector i covers columns (i TPR + t) V .. + V - 1
template <typename T, int V, int NV, int TPR>
__device__ __forceinline__ void rn_load(float (&x)[NV * V], const T* __restrict__ row, int d, int t) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    if constexpr (V == 1) {
      x[i] = c < d ? to_f32<T>(row[c]) : 0.f;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const f32x4 v = c < d ? *(const f32x4*)(row + c + q) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i * V + q + j] = v[j];
      }
    } else {
      const uint4 v = c < d ? *(const uint4*)(row + c) : make_uint4(0, 0, 0, 0);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[i * 8 + 2 * j] = __uint_as_float(w[j] << 16);
        x[i * 8 + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
}

template <typename T, int V, int NV, int TPR>
__device__ __forceinline__ void rn_store(T* __restrict__ row, const float (&x)[NV * V], int d, int t) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    if (c >= d) continue;
    if constexpr (V == 1) {
      row[c] = from_f32<T>(x[i]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int q = 0; q < V; q += 4)
        *(f32x4*)(row + c + q) = f32x4{x[i * V + q], x[i * V + q + 1], x[i * V + q + 2], x[i * V + q + 3]};
    } else {
      *(uint4*)(row + c) = make_uint4(pk_bf16(x[i * 8], x[i * 8 + 1]), pk_bf16(x[i * 8 + 2], x[i * 8 + 3]),
                                      pk_bf16(x[i * 8 + 4], x[i * 8 + 5]), pk_bf16(x[i * 8 + 6], x[i * 8 + 7]));
    }
  }
}

// sums of N values over the TPR threads of a row; every thread gets them.  TPR 256: through red, and
// the barrier behind the last read lets the next call write it.
template <int TPR, int N>
__device__ __forceinline__ void rn_sum(float (&v)[N], float* red) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = group_sum<16>(v[k]);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[k]), __float_as_uint(v[k]), false, false);
    v[k] = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]), __float_as_uint(v[k]), false, false);
    v[k] = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) red[k * 4 + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (red[k * 4] + red[k * 4 + 1]) + (red[k * 4 + 2] + red[k * 4 + 3]);
    __syncthreads();
  }
}

// mean (0 for RMS) and 1 / sqrt(variance + eps) of a row
template <int V, int NV, int TPR>
__device__ __forceinline__ void rn_stats(const float (&x)[NV * V], int d, int t, bool rms, float eps, float* red,
                                         float& mu, float& rs) {
  float s[1] = {0.f};
  if (!rms) {
#pragma unroll
    for (int e = 0; e < NV * V; ++e) s[0] += x[e];   // columns past d hold 0
    rn_sum<TPR, 1>(s, red);
  }
  mu = s[0] / d;
  float q[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * TPR + t) * V < d)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float c = x[i * V + j] - mu;
        q[0] = fmaf(c, c, q[0]);
      }
  rn_sum<TPR, 1>(q, red);
  rs = 1.0f / sqrtf(q[0] / d + eps);
}

// One row a wave (TPR 64, 4 rows a block) or a block (TPR 256).  Bound by HBM: bf16, 65536 rows of 1024: 113 us for four
// tensors, 4.7 TB/s, the rate of a large copy.
template <typename T, int V, int NV, int TPR>
__global__ void __launch_bounds__(256) resnorm_fwd_kernel(RnFwd a) {
  __shared__ float red[8];
  constexpr int E = NV * V;
  const int t = threadIdx.x & (TPR - 1), d = a.d;
  for (int64_t row = (int64_t)blockIdx.x * (256 / TPR) + (TPR == 64 ? threadIdx.x >> 6 : 0); row < a.rows;
       row += (int64_t)gridDim.x * (256 / TPR)) {
    float h[E], y[E], w[E], b[E];
    rn_load<T, V, NV, TPR>(y, (const T*)a.y + row * d, d, t);
    rn_load<T, V, NV, TPR>(h, (const T*)a.h + row * d, d, t);
    if (a.pg) {
      float mu, rs;
      rn_load<float, V, NV, TPR>(w, a.pg, d, t);
      rn_stats<V, NV, TPR>(y, d, t, a.rms, a.eps, red, mu, rs);
      if (a.pb) {
        rn_load<float, V, NV, TPR>(b, a.pb, d, t);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = fmaf((y[e] - mu) * rs, w[e], b[e]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = (y[e] - mu) * rs * w[e];
      }
      if (a.stats && t == 0) {
        a.stats[row] = mu;
        a.stats[a.rows + row] = rs;
      }
    }
    if (a.gate) {
      rn_load<T, V, NV, TPR>(w, (const T*)a.gate + (int64_t)((uint32_t)row / (uint32_t)a.gate_rows) * d, d, t);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = fmaf(a.scale, h[e], y[e]);
    // (columns past d: the weights read as 0 there, and so y and h' are 0 in the sums)
    rn_store<T, V, NV, TPR>((T*)a.ho + row * d, h, d, t);
    float mu, rs;
    rn_load<float, V, NV, TPR>(w, a.ng, d, t);
    rn_stats<V, NV, TPR>(h, d, t, a.rms, a.eps, red, mu, rs);
    if (a.nb) {
      rn_load<float, V, NV, TPR>(b, a.nb, d, t);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = fmaf((h[e] - mu) * rs, w[e], b[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = (h[e] - mu) * rs * w[e];
    }
    rn_store<T, V, NV, TPR>((T*)a.u + row * d, h, d, t);
    if (a.stats && t == 0) {
      a.stats[2 * a.rows + row] = mu;
      a.stats[3 * a.rows + row] = rs;
    }
  }
}

// Backward of a segment of rows that share a gate row, or of several gate rows' rows (a wave has whole gate rows then).  h' is
// formed again in f32 from h, y and the gate (h itself is read in the place of the stored h', whose rounding would go into the f32
// weight gradients), the column sums stay in registers over the segment and leave as one row of partial
// sums a block, which resnorm_sum_kernel adds in a fixed order.  Bound by HBM: bf16, 16 clips of 4096 rows of 1024, gate by
// clip: 191 us for six tensors, 4.2 TB/s, and 11 us of column sums.
// (Forms of their own, so that none has another's registers: bf16 rows of 1024 take two waves a SIMD, just.)
enum { RN_SEGMENT, RN_SEVERAL, RN_GATE32 };   // a segment; several gate rows; a segment that leaves each row's gate gradient in f32
template <typename T, int V, int NV, int TPR, int FORM>
__global__ void __launch_bounds__(256) resnorm_bwd_kernel(RnBwd a) {
  __shared__ float red[8];
  __shared__ float colred[TPR == 64 ? 3 * 64 * NV * V : 1];
  constexpr int E = NV * V, WAVES = 256 / TPR;
  constexpr bool SEVERAL = FORM == RN_SEVERAL;
  const RnFwd& f = a.f;
  const int t = threadIdx.x & (TPR - 1), wave = TPR == 64 ? threadIdx.x >> 6 : 0, d = f.d;
  float ng[E], pg[E], sng[E], snb[E], spg[E], spb[E], sgt[E];
  rn_load<float, V, NV, TPR>(ng, f.ng, d, t);
  if (f.pg) rn_load<float, V, NV, TPR>(pg, f.pg, d, t);
#pragma unroll
  for (int e = 0; e < E; ++e) sng[e] = snb[e] = spg[e] = spb[e] = sgt[e] = 0.f;
  // a segment, its rows dealt to the waves; SEVERAL: the wave's own gate rows, one after another
  int64_t row, end;
  int left = f.gate_rows;   // rows to the end of the gate row
  if constexpr (SEVERAL) {
    const int64_t group = blockIdx.x * a.per + wave * (a.per / WAVES);
    row = group * a.group_rows;
    end = min(group + a.per / WAVES, a.groups) * a.group_rows;
  } else {
    const int64_t group = blockIdx.x / a.segs, r0 = group * a.group_rows + (blockIdx.x % a.segs) * a.seg;
    row = r0 + wave;
    end = min(r0 + a.seg, (group + 1) * a.group_rows);
  }
  for (; row < end; row += SEVERAL ? 1 : WAVES) {
    float h[E], y[E], dt[E], du[E], gt[E];
    rn_load<T, V, NV, TPR>(y, (const T*)f.y + row * d, d, t);
    rn_load<T, V, NV, TPR>(h, (const T*)f.h + row * d, d, t);
    rn_load<T, V, NV, TPR>(du, (const T*)a.du + row * d, d, t);
    rn_load<T, V, NV, TPR>(dt, (const T*)a.dho + row * d, d, t);
    if (f.gate) rn_load<T, V, NV, TPR>(gt, (const T*)f.gate + (int64_t)((uint32_t)row / (uint32_t)f.gate_rows) * d, d, t);
    const float mu2 = f.stats[2 * f.rows + row], rs2 = f.stats[3 * f.rows + row];
    float mu1 = 0.f, rs1 = 0.f;
    if (f.pg) {
      mu1 = f.stats[row];
      rs1 = f.stats[f.rows + row];
    }
    // y := its norm before the weights (y itself without one); h := (h' - mean) / sd
    float yn[E];   // post(y)
    if (f.pg) {
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = (y[e] - mu1) * rs1;
      if (f.pb) {
        float b[E];
        rn_load<float, V, NV, TPR>(b, f.pb, d, t);
#pragma unroll
        for (int e = 0; e < E; ++e) yn[e] = fmaf(y[e], pg[e], b[e]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) yn[e] = y[e] * pg[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) yn[e] = y[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = (fmaf(f.scale, h[e], f.gate ? yn[e] * gt[e] : yn[e]) - mu2) * rs2;
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {   // columns past d: du and ng are 0
      sng[e] = fmaf(du[e], h[e], sng[e]);
      snb[e] += du[e];
      du[e] *= ng[e];
      s[0] = fmaf(du[e], h[e], s[0]);
      s[1] += du[e];
    }
    rn_sum<TPR, 2>(s, red);
    const float m2 = s[0] / d, m1 = f.rms ? 0.f : s[1] / d;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dt[e] = fmaf(rs2, du[e] - m1 - h[e] * m2, dt[e]);   // t: the whole gradient of h'
      du[e] = f.scale * dt[e];
    }
    rn_store<T, V, NV, TPR>((T*)a.dh + row * d, du, d, t);
    if (f.gate) {
      if (a.by_row) {
#pragma unroll
        for (int e = 0; e < E; ++e) du[e] = dt[e] * yn[e];
        if constexpr (FORM == RN_GATE32) rn_store<float, V, NV, TPR>((float*)a.dgate + row * d, du, d, t);
        else rn_store<T, V, NV, TPR>((T*)a.dgate + row * d, du, d, t);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) sgt[e] = fmaf(dt[e], yn[e], sgt[e]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) dt[e] *= gt[e];
    }
    if (f.pg) {
      float q[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        spg[e] = fmaf(dt[e], y[e], spg[e]);
        spb[e] += dt[e];
        dt[e] *= pg[e];   // 0 past d
        q[0] = fmaf(dt[e], y[e], q[0]);
        q[1] += dt[e];
      }
      rn_sum<TPR, 2>(q, red);
      const float n2 = q[0] / d, n1 = f.rms ? 0.f : q[1] / d;
#pragma unroll
      for (int e = 0; e < E; ++e) dt[e] = rs1 * (dt[e] - n1 - y[e] * n2);
    }
    rn_store<T, V, NV, TPR>((T*)a.dy + row * d, dt, d, t);
    if (SEVERAL && --left == 0) {
      rn_store<T, V, NV, TPR>((T*)a.dgate + (int64_t)((uint32_t)row / (uint32_t)f.gate_rows) * d, sgt, d, t);
      left = f.gate_rows;
#pragma unroll
      for (int e = 0; e < E; ++e) sgt[e] = 0.f;
    }
  }
  // the block's column sums: its waves' in order, then one row a kind
  const int64_t blocks = gridDim.x;
  auto leave = [&](float(&v)[E], int kind) {
    if constexpr (TPR == 64) {
      __syncthreads();
      if (wave)
#pragma unroll
        for (int e = 0; e < E; ++e) colred[((wave - 1) * E + e) * 64 + t] = v[e];
      __syncthreads();
      if (!wave)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = ((v[e] + colred[e * 64 + t]) + colred[(E + e) * 64 + t]) + colred[(2 * E + e) * 64 + t];
    }
    if (!wave) rn_store<float, V, NV, TPR>(a.part + (kind * blocks + blockIdx.x) * d, v, d, t);
  };
  leave(sng, 0);
  if (f.nb) leave(snb, 1);
  if (f.pg) leave(spg, 2);
  if (f.pb) leave(spb, 3);
  if (f.gate && !a.by_row && !SEVERAL) leave(sgt, 4);
}

// Column sums of the partial rows: block (x, y) adds 64 columns of list y -- one of the weights'
// over all blocks, or a gate row's over its own -- 16 rows at a time and then in a fixed tree.
struct RnSum {
  int d, lists;
  int64_t segs, blocks, gate0;  // gate0: the first list that is a gate row
  const float* part;
  float* out[4];
  int kind[4];
  void* dgate;
  int bf16;
};
__global__ void __launch_bounds__(1024) resnorm_sum_kernel(RnSum a) {
  __shared__ float red[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), ph = threadIdx.x >> 6;
  for (int64_t list = blockIdx.y; list < a.lists; list += gridDim.y) {
    const bool gate = list >= a.gate0;
    const int64_t first = gate ? (list - a.gate0) * a.segs : 0, count = gate ? a.segs : a.blocks;
    const float* p = a.part + ((gate ? 4 : a.kind[list]) * a.blocks + first) * a.d + c;
    float s = 0.f;
    if (c < a.d)
#pragma unroll 4
      for (int64_t r = ph; r < count; r += 16) s += p[r * a.d];
    red[ph][threadIdx.x & 63] = s;
    __syncthreads();
    if (ph == 0 && c < a.d) {
#pragma unroll
      for (int k = 1; k < 16; ++k) s += red[k][threadIdx.x];
      if (!gate) a.out[list][c] = s;
      else if (a.bf16) ((bf16_t*)a.dgate)[(list - a.gate0) * a.d + c] = f2bf(s);
      else ((float*)a.dgate)[(list - a.gate0) * a.d + c] = s;
    }
    __syncthreads();
  }
}

// Sums of an f32 array over some of its axes, those that a gate was broadcast along.  Neighbouring axes of one kind count as
// one; where the last is kept a lane has an output, else a wave has, so that neighbouring lanes read neighbouring elements
// either way.  Long sums are divided among blocks, whose parts gate_join_kernel adds.  Every sum has one order.  Bound
// by reading the array once.
constexpr int GS_AXES = 8;   // of each kind
struct GateSum {
  int kept, summed;                                   // axes, the last one first
  int64_t kept_size[GS_AXES], kept_step[GS_AXES], summed_size[GS_AXES], summed_step[GS_AXES];
  int64_t outs, terms, parts, blocks;                 // blocks: of 64 or 4 outputs
  bool lanes;                                         // a lane an output
};
__device__ __forceinline__ int64_t gs_at(int64_t i, int axes, const int64_t* size, const int64_t* step) {
  int64_t at = 0;
  for (int k = 0; k < axes - 1; ++k) {
    at += i % size[k] * step[k];
    i /= size[k];
  }
  return axes ? at + i * step[axes - 1] : 0;
}
template <typename T>
__global__ void __launch_bounds__(256) gate_sum_kernel(GateSum a, const float* __restrict__ src, float* __restrict__ part, T* __restrict__ out) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t each = (a.terms + a.parts - 1) / a.parts, first = blockIdx.y * each, end = min(first + each, a.terms);
  for (int64_t block = blockIdx.x; block < a.blocks; block += gridDim.x) {
    const int64_t o = block * (a.lanes ? 64 : 4) + (a.lanes ? lane : wave);
    float s = 0.f;
    if (o < a.outs) {
      const float* p = src + gs_at(o, a.kept, a.kept_size, a.kept_step);
#pragma unroll 4
      for (int64_t r = first + (a.lanes ? wave : lane); r < end; r += a.lanes ? 4 : 64) s += p[gs_at(r, a.summed, a.summed_size, a.summed_step)];
    }
    if (a.lanes) {
      __syncthreads();
      red[wave][lane] = s;
      __syncthreads();
      s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    } else {
      float v[1] = {s};
      rn_sum<64, 1>(v, nullptr);
      s = v[0];
    }
    if (o >= a.outs || (a.lanes ? wave : lane)) continue;
    if (a.parts > 1) part[blockIdx.y * a.outs + o] = s;
    else out[o] = from_f32<T>(s);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) gate_join_kernel(int64_t outs, int64_t parts, const float* __restrict__ part, T* __restrict__ out) {
  const int64_t o = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);   // a wave an output
  float s[1] = {0.f};
  if (o < outs)
    for (int64_t p = threadIdx.x & 63; p < parts; p += 64) s[0] += part[p * outs + o];
  rn_sum<64, 1>(s, nullptr);
  if (o < outs && (threadIdx.x & 63) == 0) out[o] = from_f32<T>(s[0]);
}

// 0, -1 (argument) or -2 (unsupported); the axes of one kind beside each other taken together, and 1024 blocks (of whole waves 4096, as their outputs may be few)
int gs_plan(int axes, const int64_t* sizes, const uint8_t* kept, GateSum& a) {
  a = GateSum{};
  if (axes < 0 || (axes && (!sizes || !kept))) return -1;
  a.outs = a.terms = 1;
  int64_t step = 1;
  int last = -1;
  for (int i = axes - 1; i >= 0; --i) {
    if (sizes[i] < 1 || step > INT64_MAX / sizes[i]) return -1;
    if (sizes[i] == 1) continue;
    const int k = kept[i] != 0;
    int& n = k ? a.kept : a.summed;
    if (k != last && n++ == GS_AXES) return -2;
    (k ? a.kept_size : a.summed_size)[n - 1] = k == last ? (k ? a.kept_size : a.summed_size)[n - 1] * sizes[i] : sizes[i];
    if (k != last) (k ? a.kept_step : a.summed_step)[n - 1] = step;
    if (last < 0) a.lanes = k;
    last = k;
    step *= sizes[i];
    (k ? a.outs : a.terms) *= sizes[i];
  }
  a.blocks = a.lanes ? (a.outs + 63) / 64 : (a.outs + 3) / 4;
  a.parts = std::max<int64_t>(1, std::min<int64_t>((a.lanes ? 1024 : 4096) / a.blocks, a.terms / (a.lanes ? 64 : 1024)));
  return 0;
}

bool rn_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int rn_check(const RnFwd& a, int dtype, int kind) {
  if (a.rows < 0 || a.d <= 0 || a.gate_rows < 1 || (dtype != GGD_TR_F32 && dtype != GGD_TR_BF16) ||
      (kind != GGD_TR_LAYERNORM && kind != GGD_TR_RMSNORM) || !(a.eps > 0.f) || !a.ng || (a.pb && !a.pg) ||
      (a.gate && a.rows % a.gate_rows) || (a.rows && (!a.h || !a.y || !a.ho || !a.u)))
    return -1;
  return a.d > RN_MAX_D || a.rows > RN_MAX_ROWS ? -2 : 0;
}

// Blocks of the backward pass: segments of a gate row's rows, about 1024 blocks in all (4 a CU) but at least 8 rows each, so that
// the partial sums stay a small part of the traffic.  Where there are more gate rows than that (than waves of as many blocks, where
// each wave has rows of its own), a block or wave has whole gate rows, several of them, in 1024 to 2048 blocks: bf16, a training pass
// over 200000 gate rows of 2 rows of 64 columns 3054 -> 588 us against a block a gate row, 5000 of 20 rows of 1024 602 -> 524.
struct RnSegments { int64_t group_rows, groups, seg, segs, per, blocks; };
RnSegments rn_segments(int64_t rows, int d, int64_t gate_rows, bool gate) {
  RnSegments g{};
  g.group_rows = gate && gate_rows > 1 ? gate_rows : rows;
  g.groups = rows / g.group_rows;
  const int64_t waves = d <= 1024 ? 4 : 1;   // (RN_DISPATCH: a row a wave, or a block)
  if (g.groups > 1024 * waves) {
    g.per = (g.groups + 2048 * waves - 1) / (2048 * waves) * waves;
    g.blocks = (g.groups + g.per - 1) / g.per;
    return g;
  }
  const int64_t want = std::max<int64_t>(1, 1024 / g.groups);
  g.seg = std::max<int64_t>(std::min<int64_t>(8, g.group_rows), (g.group_rows + want - 1) / want);
  g.segs = (g.group_rows + g.seg - 1) / g.seg;
  g.blocks = g.segs * g.groups;
  return g;
}

// (further arguments: more of the kernel's template arguments, from their comma on)
#define RN_DISPATCH(KERNEL, T, VMAX, vec, d, GRID, ...)                                            \
  if (vec) {                                                                                       \
    if (d <= 256 * VMAX / 4) { GRID(64, (KERNEL<T, VMAX, 1, 64 __VA_ARGS__>)); }                   \
    else if (d <= 512 * VMAX / 4 && d <= 1024) { GRID(64, (KERNEL<T, VMAX, 2, 64 __VA_ARGS__>)); } \
    else if (d <= 1024) { GRID(64, (KERNEL<T, VMAX, 16 / VMAX, 64 __VA_ARGS__>)); }                \
    else if (d <= 2048) { GRID(256, (KERNEL<T, VMAX, 8 / VMAX, 256 __VA_ARGS__>)); }               \
    else if (d <= 4096) { GRID(256, (KERNEL<T, VMAX, 16 / VMAX, 256 __VA_ARGS__>)); }              \
    else { GRID(256, (KERNEL<T, VMAX, 32 / VMAX, 256 __VA_ARGS__>)); }                             \
  } else {                                                                                         \
    if (d <= 256) { GRID(64, (KERNEL<T, 1, 4, 64 __VA_ARGS__>)); }                                 \
    else if (d <= 1024) { GRID(64, (KERNEL<T, 1, 16, 64 __VA_ARGS__>)); }                          \
    else if (d <= 4096) { GRID(256, (KERNEL<T, 1, 16, 256 __VA_ARGS__>)); }                        \
    else { GRID(256, (KERNEL<T, 1, 32, 256 __VA_ARGS__>)); }                                       \
  }

}  // namespace
}  // namespace ggd

using namespace ggd;

extern "C" {

int ggd_tr_resnorm_fwd(int64_t rows, int d, int dtype, int kind, float scale, float eps, const void* h, const void* y,
                       const void* gate, int64_t gate_rows, const float* post_g, const float* post_b, const float* pre_g,
                       const float* pre_b, void* h_out, void* u, float* stats, void* stream) {
  const RnFwd a{rows, gate_rows, d, kind, scale, eps, h, y, gate, post_g, post_b, pre_g, pre_b, h_out, u, stats};
  if (const int e = rn_check(a, dtype, kind)) return e;
  if (rows == 0) return 0;
  const bool vec = d % (dtype == GGD_TR_F32 ? 4 : 8) == 0 && rn_aligned(h) && rn_aligned(y) && rn_aligned(gate) && rn_aligned(post_g) &&
                   rn_aligned(post_b) && rn_aligned(pre_g) && rn_aligned(pre_b) && rn_aligned(h_out) && rn_aligned(u);
#define RN_GRID(TPR, K) \
  hipLaunchKernelGGL(K, dim3((unsigned)std::min<int64_t>((rows + 256 / TPR - 1) / (256 / TPR), RN_MAX_GRID)), dim3(256), 0, \
                     (hipStream_t)stream, a)
  if (dtype == GGD_TR_F32) {
    RN_DISPATCH(resnorm_fwd_kernel, float, 4, vec, d, RN_GRID)
  } else {
    RN_DISPATCH(resnorm_fwd_kernel, bf16_t, 8, vec, d, RN_GRID)
  }
#undef RN_GRID
  return hipGetLastError() == hipSuccess ? 0 : -3;
}

int64_t ggd_tr_resnorm_ws(int64_t rows, int d, int64_t gate_rows, int has_gate) {
  if (rows <= 0 || rows > RN_MAX_ROWS || d <= 0 || d > RN_MAX_D || gate_rows < 1 || (has_gate && rows % gate_rows)) return 0;
  return 5 * rn_segments(rows, d, gate_rows, has_gate).blocks * d * (int64_t)sizeof(float);
}

int ggd_tr_resnorm_bwd(int64_t rows, int d, int dtype, int kind, float scale, float eps, const void* h, const void* y,
                       const void* gate, int64_t gate_rows, const float* post_g, const float* post_b, const float* pre_g,
                       const float* pre_b, const float* stats, const void* dh_out, const void* du, void* dh, void* dy,
                       void* dgate, float* d_post_g, float* d_post_b, float* d_pre_g, float* d_pre_b, void* ws,
                       int64_t ws_bytes, void* stream) {
  const bool gate32 = kind & GGD_TR_GATE_F32;
  kind &= ~GGD_TR_GATE_F32;
  RnBwd a{};
  a.f = RnFwd{rows, gate_rows, d, kind, scale, eps, h, y, gate, post_g, post_b, pre_g, pre_b, dh, dy, (float*)stats};
  a.dho = dh_out, a.du = du, a.dh = dh, a.dy = dy, a.dgate = dgate, a.part = (float*)ws;
  if (const int e = rn_check(a.f, dtype, kind)) return e;
  if (rows == 0 || (gate32 && (!gate || gate_rows != 1)) || !stats || !dh_out || !du || !gate != !dgate || !d_pre_g || !pre_b != !d_pre_b || !post_g != !d_post_g ||
      !post_b != !d_post_b)
    return -1;
  if (!ws || !rn_aligned(ws) || ws_bytes < ggd_tr_resnorm_ws(rows, d, gate_rows, gate != nullptr)) return -1;
  const RnSegments g = rn_segments(rows, d, gate_rows, gate);
  a.seg = g.seg, a.segs = g.segs, a.per = g.per, a.groups = g.groups, a.group_rows = g.group_rows;
  a.by_row = gate && gate_rows == 1;
  const bool vec = d % (dtype == GGD_TR_F32 ? 4 : 8) == 0 && rn_aligned(h) && rn_aligned(y) && rn_aligned(gate) && rn_aligned(post_g) &&
                   rn_aligned(post_b) && rn_aligned(pre_g) && rn_aligned(pre_b) && rn_aligned(dh_out) && rn_aligned(du) &&
                   rn_aligned(dh) && rn_aligned(dy) && rn_aligned(dgate);
  hipStream_t s = (hipStream_t)stream;
#define RN_GRID(TPR, K) hipLaunchKernelGGL(K, dim3((unsigned)g.blocks), dim3(256), 0, s, a)
  if (dtype == GGD_TR_F32) {
    if (g.per) { RN_DISPATCH(resnorm_bwd_kernel, float, 4, vec, d, RN_GRID, , RN_SEVERAL) }
    else { RN_DISPATCH(resnorm_bwd_kernel, float, 4, vec, d, RN_GRID, , RN_SEGMENT) }   // (whose gate gradients are f32 anyway)
  } else {
    if (g.per) { RN_DISPATCH(resnorm_bwd_kernel, bf16_t, 8, vec, d, RN_GRID, , RN_SEVERAL) }
    else if (gate32) { RN_DISPATCH(resnorm_bwd_kernel, bf16_t, 8, vec, d, RN_GRID, , RN_GATE32) }
    else { RN_DISPATCH(resnorm_bwd_kernel, bf16_t, 8, vec, d, RN_GRID, , RN_SEGMENT) }
  }
#undef RN_GRID
  RnSum r{};
  r.d = d, r.blocks = g.blocks, r.segs = g.segs, r.part = a.part, r.dgate = dgate, r.bf16 = dtype == GGD_TR_BF16;
  float* const out[4] = {d_pre_g, d_pre_b, d_post_g, d_post_b};
  for (int k = 0; k < 4; ++k)
    if (out[k]) {
      r.out[r.gate0] = out[k];
      r.kind[r.gate0++] = k;
    }
  r.lists = r.gate0 + (gate && !a.by_row && !g.per ? g.groups : 0);
  hipLaunchKernelGGL(resnorm_sum_kernel, dim3((d + 63) / 64, (unsigned)std::min<int64_t>(r.lists, 65535)), dim3(1024), 0, s, r);
  return hipGetLastError() == hipSuccess ? 0 : -3;
}

int64_t ggd_tr_gate_sum_ws(int axes, const int64_t* sizes, const uint8_t* kept) {
  GateSum a;
  return gs_plan(axes, sizes, kept, a) || a.parts == 1 ? 0 : a.parts * a.outs * (int64_t)sizeof(float);
}

int ggd_tr_gate_sum(int axes, const int64_t* sizes, const uint8_t* kept, const float* src, int dtype, void* out, void* ws, int64_t ws_bytes,
                    void* stream) {
  GateSum a;
  if (const int e = gs_plan(axes, sizes, kept, a)) return e;
  if (!src || !out || (dtype != GGD_TR_F32 && dtype != GGD_TR_BF16)) return -1;
  if (a.parts > 1 && (!ws || ws_bytes < a.parts * a.outs * (int64_t)sizeof(float))) return -1;
  const dim3 grid((unsigned)std::min(a.blocks, RN_MAX_GRID), (unsigned)a.parts), join((unsigned)((a.outs + 3) / 4));
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == GGD_TR_F32) {
    hipLaunchKernelGGL(gate_sum_kernel<float>, grid, dim3(256), 0, s, a, src, (float*)ws, (float*)out);
    if (a.parts > 1) hipLaunchKernelGGL(gate_join_kernel<float>, join, dim3(256), 0, s, a.outs, a.parts, (const float*)ws, (float*)out);
  } else {
    hipLaunchKernelGGL(gate_sum_kernel<bf16_t>, grid, dim3(256), 0, s, a, src, (float*)ws, (bf16_t*)out);
    if (a.parts > 1) hipLaunchKernelGGL(gate_join_kernel<bf16_t>, join, dim3(256), 0, s, a.outs, a.parts, (const float*)ws, (bf16_t*)out);
  }
  return hipGetLastError() == hipSuccess ? 0 : -3;
}

}  // extern "C"
