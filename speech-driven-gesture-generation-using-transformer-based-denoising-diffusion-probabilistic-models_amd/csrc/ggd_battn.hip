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
int prepare(const ggd_tr_battn_args* in, BtArgs& a) {
  if (!in) return -1;
  (ggd_tr_battn_args&)a = *in;
  if (a.n < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.lq < 1 || a.lk < 1 || a.dk < 1 ||
      (a.dtype != GGD_TR_F32 && a.dtype != GGD_TR_BF16) || !(a.scale > 0.f) || !(a.scale <= 1e30f))
    return -1;
  if (a.ldq < 0 || a.ldk < 0 || a.ldv < 0 || a.ldo < 0 || a.bq < 0 || a.bk < 0 || a.bv < 0 || a.bo < 0 || a.bmask < 0 || a.bq_mask < 0) return -1;
  if (!a.table != !a.buckets || (a.table && (a.n_buckets < 1 || a.distance < 1))) return -1;
  if (a.dk > BT_MAX_DK || a.lq > BT_MAX_ROWS || a.lk > BT_MAX_ROWS || (a.table && (a.n_buckets > BT_MAX_BUCKETS || a.distance > BT_MAX_DISTANCE)))
    return -2;
  if (!a.table) a.distance = 0, a.n_buckets = 0;
  a.group = a.heads / a.kv_heads;
  if ((int64_t)a.group * a.lq > INT32_MAX - 64 ||
      (int64_t)a.n * a.heads * ((std::max(a.lq, a.lk) + 31) / 32) > (1 << 24) - 8)
    return -2;   // rows of a kv head; threads of a launch (256 a block, and an axis is divided only where there are few blocks)
  a.off = (int)std::max<int64_t>(-(1 << 30), std::min<int64_t>(1 << 30, a.offset));
  a.c = a.scale * BT_LOG2E;
  a.splits = 1;
  return 0;
}

size_t esize(const BtArgs& a) { return a.dtype == GGD_TR_F32 ? 4 : 2; }

// 16-byte loads of rows: every row starts at a multiple of 16 bytes and holds whole units
bool vec_rows(const BtArgs& a, const void* p, int64_t ld, int64_t b) {
  const int64_t per = 16 / (int64_t)esize(a);
  return aligned(p, 16) && ld % per == 0 && b % per == 0 && a.dk % per == 0;
}

// Few rows: the rows of a kv head's query heads fill one MFMA tile (32), or the tiled kernel's blocks of 128
// rows of a head would leave most of the chip idle while the keys are long enough to divide among blocks.
bool few_rows(const BtArgs& a) {
  const int64_t rows = (int64_t)a.group * a.lq, blocks = (int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS);
  return rows <= 32 || (blocks < 128 && a.lk >= 512 && a.lk >= 4 * a.lq);
}

// parts of a streamed axis of `tiles` tiles so that `blocks` blocks become about 512 (2 a CU), each with at least `least` tiles
int parts(int64_t blocks, int64_t tiles, int64_t least) {
  const int64_t want = (512 + blocks - 1) / std::max<int64_t>(1, blocks);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, 64), tiles / least));
}
int few_splits(const BtArgs& a) {
  const int64_t blocks = (int64_t)a.n * a.kv_heads * (((int64_t)a.group * a.lq + 31) / 32);
  return parts(blocks, (a.lk + 31) / 32, 8);
}
int tile(const BtArgs& a) { return a.dtype == GGD_TR_F32 && a.dk > 64 ? 32 : 64; }
int dq_splits(const BtArgs& a) {
  return parts((int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS), (a.lk + tile(a) - 1) / tile(a), 4);
}
int dkv_splits(const BtArgs& a) {
  return parts((int64_t)a.n * a.kv_heads * ((a.lk + BT_ROWS - 1) / BT_ROWS), (int64_t)a.group * ((a.lq + tile(a) - 1) / tile(a)), 4);
}
int dk_class(const BtArgs& a) { return a.dk <= 32 ? 32 : a.dk <= 64 ? 64 : 128; }

int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// the backward workspace: delta, the blocks' table gradients (bf16: two lists, and BtArgs::rest), then the parts of dq and
// later of dk and dv
struct Space { int64_t delta, table, rest, part; };
Space backward_space(const BtArgs& a) {
  Space s;
  s.delta = up((int64_t)a.n * a.heads * a.lq * 4);
  const int ds = dq_splits(a), ks = dkv_splits(a);
  const int two = a.dtype == GGD_TR_BF16;
  s.table = a.dtable ? up((int64_t)a.n * a.heads * ((a.lq + BT_ROWS - 1) / BT_ROWS) * (ds + two) * a.n_buckets * 4) : 0;
  s.rest = a.dtable && two ? up(2 * ds * (int64_t)a.n * a.heads * a.lq * 4) : 0;
  const int64_t pq = ds > 1 ? (int64_t)ds * a.n * a.lq * a.heads * a.dk * 4 : 0;
  const int64_t pk = ks > 1 ? 2 * (int64_t)ks * a.n * a.lk * a.kv_heads * a.dk * 4 : 0;
  s.part = up(std::max(pq, pk));
  return s;
}
int64_t forward_space(const BtArgs& a) {
  if (!few_rows(a)) return 0;
  const int s = few_splits(a);
  if (s == 1) return 0;
  const int64_t rows = ((int64_t)a.group * a.lq + 31) / 32 * 32 * a.n * a.kv_heads;
  return up(rows * s * (dk_class(a) + 4) * 4);
}

const Launch& launch(const BtArgs& a) { return a.dtype == GGD_TR_F32 ? battn_f32(a) : pick<bf16_t>(a); }

}  // namespace
}  // namespace battn
}  // namespace ggd

using namespace ggd;
using namespace ggd::battn;

extern "C" {

int64_t ggd_tr_battn_ws(const ggd_tr_battn_args* args, int backward) {
  BtArgs a{};
  if (prepare(args, a) || a.n == 0) return 0;
  if (!backward) return forward_space(a);
  const Space s = backward_space(a);
  return s.delta + s.table + s.rest + s.part;
}

int ggd_tr_battn_fwd(const ggd_tr_battn_args* args, void* stream) {
  BtArgs a{};
  if (const int e = prepare(args, a)) return e;
  if (a.n == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.o || !a.stat != !a.o32) return -1;
  const int64_t need = forward_space(a);
  if (need && (!a.ws || !aligned(a.ws, 16) || a.ws_bytes < need)) return -1;
  a.vec = vec_rows(a, a.q, a.ldq, a.bq) && vec_rows(a, a.k, a.ldk, a.bk) && vec_rows(a, a.v, a.ldv, a.bv);
  a.vec_o = a.dk % 4 == 0 && a.ldo % 4 == 0 && a.bo % 4 == 0 && aligned(a.o, 4 * esize(a)) && aligned(a.o32, 16);
  if (!aligned(a.stat, 8)) return -1;
  if (few_rows(a)) {
    a.splits = few_splits(a);
    a.part = (float*)a.ws;
    return launch(a).few(a, (hipStream_t)stream) == hipSuccess ? 0 : -3;
  }
  return launch(a).fwd(a, (hipStream_t)stream) == hipSuccess ? 0 : -3;
}

int ggd_tr_battn_bwd(const ggd_tr_battn_args* args, void* stream) {
  BtArgs a{};
  if (const int e = prepare(args, a)) return e;
  if (a.n == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.stat || !a.o32 || !a.dout || !a.dq || !a.dk_out || !a.dv || (a.dtable && !a.table)) return -1;
  const Space s = backward_space(a);
  if (!a.ws || !aligned(a.ws, 16) || a.ws_bytes < s.delta + s.table + s.rest + s.part || !aligned(a.stat, 8)) return -1;
  a.delta = (float*)a.ws;
  a.dtab = (float*)((char*)a.ws + s.delta);
  a.rest = (float*)((char*)a.ws + s.delta + s.table);
  a.part = (float*)((char*)a.ws + s.delta + s.table + s.rest);
  const int64_t ldo = (int64_t)a.heads * a.dk;
  a.vec = vec_rows(a, a.q, a.ldq, a.bq) && vec_rows(a, a.k, a.ldk, a.bk) && vec_rows(a, a.v, a.ldv, a.bv) && vec_rows(a, a.dout, ldo, ldo);
  a.vec_o = a.dk % 4 == 0 && aligned(a.dq, 4 * esize(a)) && aligned(a.dk_out, 4 * esize(a)) && aligned(a.dv, 4 * esize(a));
  a.splits = dq_splits(a);
  if (launch(a).dq(a, (hipStream_t)stream) != hipSuccess) return -3;
  a.splits = dkv_splits(a);
  return launch(a).dkv(a, (hipStream_t)stream) == hipSuccess ? 0 : -3;
}

}  // extern "C"
