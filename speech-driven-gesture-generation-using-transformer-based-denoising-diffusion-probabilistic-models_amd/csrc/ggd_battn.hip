// ggd_battn.hip -- entry points of the training path's attention for any lengths (include/ggd_train.h,
// ggd_tr_battn_*) and its kernels on bf16 rows; ggd_battn.h has the mathematics, ggd_battn_f32.hip the f32 kernels.
#include "ggd_battn_kernels.h"

namespace ggd {
namespace battn {
const Launch& battn_f32(const BtArgs& a);   // ggd_battn_f32.hip

namespace {

constexpr int BT_MAX_ROWS = 1 << 28;   // rows and keys: positions and distances fit 32 bits

bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// 0, -1 (argument) or -2 (unsupported), and the launch-side fields
int prepare(const ggd_tr_battn_args* in, BtArgs& a, bool backward) {
  if (!in) return -1;
  (ggd_tr_battn_args&)a = *in;
  if (a.n < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.lq < 1 || a.lk < 1 || a.dk < 1 ||
      (a.dtype != GGD_TR_F32 && a.dtype != GGD_TR_BF16) || !(a.scale > 0.f) || !(a.scale <= 1e30f))
    return -1;
  if (a.ldq < 0 || a.ldk < 0 || a.ldv < 0 || a.ldo < 0 || a.bq < 0 || a.bk < 0 || a.bv < 0 || a.bo < 0 || a.bmask < 0 || a.bq_mask < 0) return -1;
  if (!a.table != !a.buckets || (a.table && (a.n_buckets < 1 || a.distance < 1))) return -1;
  if (a.dk > BT_MAX_DK || a.lq > BT_MAX_ROWS || a.lk > BT_MAX_ROWS || (a.table && (a.n_buckets > BT_MAX_BUCKETS || a.distance > BT_MAX_DISTANCE)))
    return -2;
  // rows that are packed lie their own width apart, and a tile of 64 of them is read by 32-bit byte offsets
  const int64_t head_bytes = (a.dk * (a.dtype == GGD_TR_F32 ? 4 : 2) + 15) / 16 * 16;
  if ((63 * (int64_t)a.heads + 1) * head_bytes > INT32_MAX) return -2;
  if (!a.table) a.distance = 0, a.n_buckets = 0;
  a.group = a.heads / a.kv_heads;
  if ((int64_t)a.group * a.lq > INT32_MAX - 64 || (int64_t)a.n * a.heads > 1 << 22 || (int64_t)a.heads * a.n_buckets > 1 << 25 ||
      (int64_t)a.n * a.heads * ((a.lq + 31) / 32) > 1 << 22)
    return -2;   // rows of a kv head; threads of a launch (256 a block, 64 a table entry; an axis is divided only where there are few blocks)
  // ... and 512 a block of 128 keys in the backward pass, where one follows; the forward pass has no block a key
  if ((backward || a.stat) && (int64_t)a.n * a.kv_heads * ((a.lk + BT_ROWS - 1) / BT_ROWS) > 1 << 22) return -2;
  a.off = (int)std::max<int64_t>(-(1 << 30), std::min<int64_t>(1 << 30, a.offset));
  a.c = a.scale * BT_LOG2E;
  a.splits = 1;
  return 0;
}

size_t esize(const BtArgs& a) { return a.dtype == GGD_TR_F32 ? 4 : 2; }

// The kernels read rows in 16-byte units, and a tile of 64 rows by 32-bit offsets: rows that do not start at a multiple of 16
// bytes, hold other than whole units or lie too far apart are packed first (one more pass over them, without a limit on strides;
// prepare() has one on their width).
constexpr int64_t BT_MAX_LD = 1 << 22;
bool whole_rows(const BtArgs& a, const void* p, int64_t ld, int64_t b) {
  const int64_t per = 16 / (int64_t)esize(a);
  return aligned(p, 16) && ld % per == 0 && ld <= BT_MAX_LD && b % per == 0 && a.dk % per == 0;
}
int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }
// bytes of each operand's packed rows, 0 where it is read in place: an operand out of line is packed alone (a stream's new query does not
// copy its memory), but where dk itself is no whole units all are
struct Packed {
  int64_t q, k, v, dout;
  int64_t all() const { return q + k + v + dout; }
};
Packed packed_space(const BtArgs& a, bool backward) {
  const int64_t per = 16 / (int64_t)esize(a), row = (a.dk + per - 1) / per * 16, ldo = (int64_t)a.heads * a.dk;
  const int64_t q = up((int64_t)a.n * a.lq * a.heads * row), k = up((int64_t)a.n * a.lk * a.kv_heads * row);
  return {whole_rows(a, a.q, a.ldq, a.bq) ? 0 : q, whole_rows(a, a.k, a.ldk, a.bk) ? 0 : k, whole_rows(a, a.v, a.ldv, a.bv) ? 0 : k,
          !backward || whole_rows(a, a.dout, ldo, ldo) ? 0 : q};
}

// Few rows: the rows of a kv head's query heads fit one MFMA tile (32), or the call is small beside the keys it reads and the tiled
// kernel's blocks of 128 rows would not fill the chip.  Blocks of 32 rows start sooner and divide finer: bf16, 8 heads of 64,
// 128 rows over 16384 keys 32 us for the tiled kernel's 50, f32, 2 heads, 256 over 4096 25 for 35.  Past 2^24 scores they read each
// key too often: bf16, 8 heads of 128, 1000 rows over 16000 297 us for 95, f32, 2 heads of 64, 4000 over 16000 442 for 327; and f32
// heads past 64, of one wave a SIMD, past 2^22: 8 heads of 128, 256 over 4096 132 us for 73.
bool few_rows(const BtArgs& a) {
  const int64_t rows = (int64_t)a.group * a.lq, blocks = (int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS);
  const int64_t scores = a.dtype == GGD_TR_F32 && a.dk > 64 ? 1 << 22 : 1 << 24;
  return rows <= 32 || (blocks < 128 && a.lk >= 512 && a.lk >= 4 * a.lq && (int64_t)a.n * a.heads * a.lq <= scores / a.lk);
}

// bf16 weights and ds, rounded once for their products, are off by up to 2^-8 each: a result's own rounding again, and over few
// keys more in dq, where the roundings of o's weights do not average out in delta = do . o.  Where the call is small, or reads
// its keys for few rows, a second product of what the rounding left costs little (few rows up to 32 are bound by their keys, more of them
// up to 7 % of a training pass's kernels: 86 -> 92 us for 8 heads of 64, 256 rows over 8192): 27 -> 30 us at 16 clips x 8 heads, 128 x 128
// (whose host side takes 70), 485 -> 523 at 256 clips x 8 heads, 500 over 64 keys; above it stays one, 81 -> 98 us at 8 x 16 heads, 512 x 512.
bool fine_weights(const BtArgs& a) {
  return a.dtype == GGD_TR_BF16 && (few_rows(a) || a.lk <= 64 || (int64_t)a.n * a.heads * a.lq <= (1 << 22) / a.lk);
}

// Parts of a streamed axis of `tiles` tiles: the fewest whose rounds of blocks over the chip's `slots` take (nearly) the least time,
// each part with at least `least` tiles, at most 64 of them.
int parts(int64_t blocks, int64_t tiles, int64_t least, int64_t slots) {
  int best = 1;
  double time = (double)((blocks + slots - 1) / slots);
  for (int64_t s = 2; s <= std::min<int64_t>(64, tiles / least); ++s) {
    const double t = (double)((blocks * s + slots - 1) / slots) / s;
    if (t < 0.93 * time) best = (int)s, time = t;
  }
  return best;
}
// blocks that run at once: 256 CUs, and as many a CU as the kernel has waves a SIMD
int64_t slots(const BtArgs& a, int bf16_dk, int f32_dk) { return a.dk <= (a.dtype == GGD_TR_BF16 ? bf16_dk : f32_dk) ? 512 : 256; }
int few_splits(const BtArgs& a) {
  const int64_t blocks = (int64_t)a.n * a.kv_heads * (((int64_t)a.group * a.lq + 31) / 32);
  return parts(blocks, (a.lk + 31) / 32, 8, slots(a, 64, 32));
}
int tile(const BtArgs& a) { return a.dtype == GGD_TR_F32 && a.dk > 64 ? 32 : 64; }
int fwd_splits(const BtArgs& a) {
  if (few_rows(a)) return few_splits(a);
  return parts((int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS), (a.lk + tile(a) - 1) / tile(a), 4, slots(a, 128, 64));
}
int dq_splits(const BtArgs& a) {
  return parts((int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS), (a.lk + tile(a) - 1) / tile(a), 4, slots(a, 128, 64));
}
int dkv_splits(const BtArgs& a) {
  return parts((int64_t)a.n * a.kv_heads * ((a.lk + BT_ROWS - 1) / BT_ROWS), (int64_t)a.group * ((a.lq + tile(a) - 1) / tile(a)), 4,
               slots(a, 64, 32));
}
int dk_class(const BtArgs& a) { return a.dk <= 32 ? 32 : a.dk <= 64 ? 64 : 128; }

// the backward workspace: packed rows, delta, the blocks' table gradients (bf16: two lists, and BtArgs::rest), then the parts of dq and
// later of dk and dv
struct Space {
  int64_t pack, delta, table, rest, part;
  int64_t all() const { return pack + delta + table + rest + part; }
};
Space backward_space(const BtArgs& a) {
  Space s;
  s.pack = packed_space(a, true).all();
  s.delta = up((int64_t)a.n * a.heads * a.lq * 4);
  const int ds = dq_splits(a), ks = dkv_splits(a);
  const int two = a.dtype == GGD_TR_BF16;
  s.table = a.dtable ? up((int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS) * (ds + two) * a.n_buckets * 4) : 0;
  s.rest = a.dtable && two ? up(2 * ds * (int64_t)a.n * a.heads * a.lq * 4) : 0;
  const int64_t pq = ds > 1 ? (int64_t)ds * a.n * a.lq * a.heads * a.dk * 4 : 0;
  const int64_t pk = ks > 1 && a.dk_out ? 2 * (int64_t)ks * a.n * a.lk * a.kv_heads * a.dk * 4 : 0;
  s.part = up(std::max(pq, pk));
  return s;
}
Space forward_space(const BtArgs& a) {
  Space s{};
  s.pack = packed_space(a, false).all();
  if (const int splits = fwd_splits(a); splits > 1)
    s.part = up(((int64_t)a.group * a.lq + 31) / 32 * 32 * a.n * a.kv_heads * splits * (dk_class(a) + 4) * 4);
  return s;
}

const Launch& launch(const BtArgs& a) { return a.dtype == GGD_TR_F32 ? battn_f32(a) : pick<bf16_t>(a); }

// q, k, v (and dout) as the kernels read them, packed into the workspace's first part where they have to be
hipError_t rows(BtArgs& a, bool backward, hipStream_t s) {
  const Packed p = packed_space(a, backward);
  const int64_t per = 16 / (int64_t)esize(a), dkp = (a.dk + per - 1) / per * per;
  char* at = (char*)a.ws;
  const Launch& l = launch(a);
  auto pack = [&](int64_t bytes, const void*& src, int64_t& ld, int64_t& b, int rows, int heads) {
    if (!bytes) return hipSuccess;
    const hipError_t e = l.pack(a, src, ld, b, rows, heads, at, s);
    src = at, ld = heads * dkp, b = rows * ld;
    at += bytes;
    return e;
  };
  int64_t bdo = a.lq * (a.lddo = (int64_t)a.heads * a.dk);
  if (const hipError_t e = pack(p.q, a.q, a.ldq, a.bq, a.lq, a.heads)) return e;
  if (const hipError_t e = pack(p.k, a.k, a.ldk, a.bk, a.lk, a.kv_heads)) return e;
  if (const hipError_t e = pack(p.v, a.v, a.ldv, a.bv, a.lk, a.kv_heads)) return e;
  if (const hipError_t e = pack(p.dout, a.dout, a.lddo, bdo, a.lq, a.heads)) return e;
  a.hq = a.hk = dkp;   // (dk where one is read in place)
  return hipSuccess;
}

}  // namespace
}  // namespace battn
}  // namespace ggd

using namespace ggd;
using namespace ggd::battn;

extern "C" {

int64_t ggd_tr_battn_ws(const ggd_tr_battn_args* args, int backward) {
  BtArgs a{};
  if (prepare(args, a, backward) || a.n == 0) return 0;
  return (backward ? backward_space(a) : forward_space(a)).all();
}

int ggd_tr_battn_fwd(const ggd_tr_battn_args* args, void* stream) {
  BtArgs a{};
  if (const int e = prepare(args, a, false)) return e;
  if (a.n == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.o || !a.stat != !a.o32) return -1;
  const Space space = forward_space(a);
  if (space.all() && (!a.ws || !aligned(a.ws, 16) || a.ws_bytes < space.all())) return -1;
  if (!aligned(a.stat, 8)) return -1;
  a.vec_o = a.dk % 4 == 0 && a.ldo % 4 == 0 && a.bo % 4 == 0 && aligned(a.o, 4 * esize(a)) && aligned(a.o32, 16);
  const bool few = few_rows(a);
  a.splits = fwd_splits(a);
  a.fine = fine_weights(a);
  a.part = (float*)((char*)a.ws + space.pack);
  const hipStream_t s = (hipStream_t)stream;
  if (rows(a, false, s) != hipSuccess) return -3;
  return (few ? launch(a).few(a, s) : launch(a).fwd(a, s)) == hipSuccess ? 0 : -3;
}

int ggd_tr_battn_bwd(const ggd_tr_battn_args* args, void* stream) {
  BtArgs a{};
  if (const int e = prepare(args, a, true)) return e;
  if (a.n == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.stat || !a.o32 || !a.dout || !a.dq || !a.dk_out != !a.dv || (a.dtable && !a.table)) return -1;
  const Space space = backward_space(a);
  if (!a.ws || !aligned(a.ws, 16) || a.ws_bytes < space.all() || !aligned(a.stat, 8) || !aligned(a.o32, a.dk % 4 ? 4 : 16)) return -1;
  char* at = (char*)a.ws + space.pack;
  a.delta = (float*)at;
  a.dtab = (float*)(at + space.delta);
  a.rest = (float*)(at + space.delta + space.table);
  a.part = (float*)(at + space.delta + space.table + space.rest);
  a.vec_o = a.dk % 4 == 0 && aligned(a.dq, 4 * esize(a)) && aligned(a.dk_out, 4 * esize(a)) && aligned(a.dv, 4 * esize(a));
  a.fine = fine_weights(a);
  const int dqs = dq_splits(a), dkvs = dkv_splits(a);
  const hipStream_t s = (hipStream_t)stream;
  if (rows(a, true, s) != hipSuccess) return -3;
  a.splits = dqs;
  if (launch(a).dq(a, s) != hipSuccess) return -3;
  if (!a.dk_out) return 0;
  a.splits = dkvs;
  return launch(a).dkv(a, s) == hipSuccess ? 0 : -3;
}

}  // extern "C"
