"""Operators of a decoder block beyond the reference's: attention for any lengths and padded batches,
attention with a learned relative position bias, and the norms around a block fused with its gate and
residual scale.

They stand beside training.py's operators (linear, layer_norm, squared_relu, ...) and take the same token
matrices, (n, L, heads dk) rows of heads; each is hand-written HIP kernels behind include/ggd_train.h, forward
and backward, in f32 or bf16 with sums, softmax and statistics in f32.  Under torch.no_grad() a call
keeps nothing for a backward pass.  Gradients come once: a second derivative raises.  Everything is issued on the
current stream of the inputs' device, with workspaces from torch's allocator, so that calls on several
streams and captured graphs share nothing; a pass that was run once may be captured.

A wrong shape, type or device raises ValueError before anything is launched.
"""
import ctypes
import math
import struct

import torch as th
from torch.autograd.function import once_differentiable

from . import native

MAX_HEAD_DIM, MAX_BUCKETS, MAX_DISTANCE, MAX_NORM_DIM = 128, 1024, 2047, 8192   # include/ggd_train.h
_DTYPES = {th.float32: 0, th.bfloat16: 1}   # GGD_TR_F32, GGD_TR_BF16


def _ok(rc, what):
    if rc == native.GGD_ERR_UNSUPPORTED:
        raise ValueError(f"{what}: unsupported shape")
    if rc != 0:
        raise native.GgdError(f"{what} failed (ggd_train status {rc})")


def _p(t):
    return t.data_ptr() if t is not None else None


def _call(fn, args, device, what):
    """An entry point on the current stream of a device, which is the current one meanwhile."""
    stream = th._C._cuda_getCurrentRawStream(device.index)
    if device.index == th.cuda.current_device():
        rc = fn(*args, stream)
    else:
        with th.cuda.device(device):
            rc = fn(*args, stream)
    if rc != 0:
        _ok(rc, what)


def _tensors(what, first, rest):
    """All on the first one's GPU."""
    if not (isinstance(first, th.Tensor) and first.is_cuda):
        raise ValueError(f"{what}: the inputs have to be on a GPU device (no CPU fallback)")
    device = first.device
    for name, t in rest:
        if t is not None and not (isinstance(t, th.Tensor) and t.device == device):
            raise ValueError(f"{what}: {name} has to be a tensor on {device}")


def _workspace(nbytes, device):
    return th.empty(nbytes, dtype=th.uint8, device=device) if nbytes else None


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
class RelativeBuckets:
    """The bucket of each relative position d = key position - query position, the plan that a model keeps beside
    its bias table of n_buckets rows.

    With both_sides the first half of the buckets is for keys at or behind the query, the second for
    those ahead; without, all are for keys behind and those ahead share bucket 0.  A side of s buckets gives
    distances below s / 2 one bucket each; bucket s / 2 + k starts where
    |d| >= (s / 2) (max_distance / (s / 2)) ^ (k / (s - s / 2)) over the reals (compared in whole numbers,
    so that no logarithm rounds at a border), and distances from max_distance on share the last.
    """

    def __init__(self, n_buckets=32, max_distance=128, both_sides=True, device="cuda"):
        n_buckets, max_distance = int(n_buckets), int(max_distance)
        side = n_buckets // 2 if both_sides else n_buckets
        if not 1 <= n_buckets <= MAX_BUCKETS or (both_sides and n_buckets % 2) or side < 2:
            raise ValueError(f"RelativeBuckets: n_buckets {n_buckets}: up to {MAX_BUCKETS}, at least 2 a side, even with both sides")
        if not side // 2 < max_distance <= MAX_DISTANCE:
            raise ValueError(f"RelativeBuckets: max_distance {max_distance}: more than {side // 2}, up to {MAX_DISTANCE}")
        self.n_buckets, self.max_distance, self.both_sides = n_buckets, max_distance, bool(both_sides)
        near, steps, of = side // 2, side - side // 2, []
        passed = 0
        for d in range(max_distance + 1):
            if d < near:
                of.append(d)
                continue
            while passed + 1 < steps and d ** steps >= near ** (steps - passed - 1) * max_distance ** (passed + 1):
                passed += 1
            of.append(near + passed)
        behind = [of[d] for d in range(max_distance, 0, -1)]
        ahead = [side + of[d] if both_sides else 0 for d in range(1, max_distance + 1)]
        self.buckets = th.tensor(behind + [of[0]] + ahead, dtype=th.int32)   # of d = -max_distance .. max_distance
        self._on = {}
        if th.device(device).type != "cpu":
            self.on(th.device(device))

    def on(self, device):
        """The buckets on a device, copied there once."""
        device = th.device(device)
        if device.type == "cuda" and device.index is None:
            device = th.device("cuda", th.cuda.current_device())
        if device not in self._on:
            self._on[device] = self.buckets.to(device)
        return self._on[device]


def _rows(t):
    """(n, L, W) with contiguous rows: the tensor where its rows are, whatever their strides, else a copy."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _mask_rows(m):
    return m if m is None or m.stride(1) == 1 or m.shape[1] == 1 else m.contiguous()


_PACK = struct.Struct("@" + "".join({ctypes.c_int32: "i", ctypes.c_float: "f", ctypes.c_int64: "q", ctypes.c_void_p: "P"}[t]
                                    for _, t in native.BattnArgs._fields_)).pack   # ggd_tr_battn_args as bytes


def _launch(entry, inputs, geo, o=None, stat=None, o32=None, grads=(None,) * 5):
    """ggd_tr_battn_fwd or _bwd over its workspace.  grads: dout, dq, dk, dv, dtable."""
    q, k, v, table, mask, q_mask, lut = inputs
    heads, kv_heads, scale, offset = geo
    n, lq, width = q.shape
    address = lambda t: t.data_ptr() if t is not None else 0
    head = (n, heads, kv_heads, lq, k.shape[1], width // heads, _DTYPES[q.dtype], scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), address(o),
            q.stride(1), q.stride(0), k.stride(1), k.stride(0), v.stride(1), v.stride(0), width, lq * width,
            address(mask), address(q_mask), 0 if mask is None else mask.stride(0), 0 if q_mask is None else q_mask.stride(0),
            address(table), address(lut), *((0, 0, 0) if table is None else (table.shape[0], lut.shape[0] // 2, offset)),
            address(stat), address(o32), *map(address, grads))
    lib = native.load()
    backward = entry == "ggd_tr_battn_bwd"
    nbytes = lib.ggd_tr_battn_ws(_PACK(*head, 0, 0), backward)
    ws = _workspace(nbytes, q.device)
    _call(getattr(lib, entry), (_PACK(*head, address(ws), nbytes),), q.device, "attention backward" if backward else "attention")


def _attend(inputs, geo, keep):
    """o, and with keep what the backward pass needs: (stat, o32)."""
    q = inputs[0]
    n, lq, width = q.shape
    o = th.empty((n, lq, width), dtype=q.dtype, device=q.device)
    if o.numel() == 0 or inputs[1].shape[1] == 0:
        return o.zero_(), None, None
    stat = o32 = None
    if keep:
        stat = th.empty((n, geo[0], lq, 2), dtype=th.float32, device=q.device)
        o32 = o if q.dtype == th.float32 else th.empty((n, lq, width), dtype=th.float32, device=q.device)
    _launch("ggd_tr_battn_fwd", inputs, geo, o, stat, o32)
    return o, stat, o32


class _Battn(th.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, mask, q_mask, lut, geo):
        inputs = (q, k, v, table, mask, q_mask, lut)
        o, stat, o32 = _attend(inputs, geo, True)
        ctx.save_for_backward(*inputs, stat, o32)
        ctx.geo = geo
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        *inputs, stat, o32 = ctx.saved_tensors
        q, k, v, table = inputs[:4]
        new = lambda t: th.empty(t.shape, dtype=t.dtype, device=t.device)
        dq, dk, dv = new(q), new(k), new(v)
        dtable = new(table) if table is not None and ctx.needs_input_grad[3] else None
        if stat is None:   # no query, or no key
            return (*(t if t is None else t.zero_() for t in (dq, dk, dv, dtable)), None, None, None, None)
        do = do.contiguous()
        _launch("ggd_tr_battn_bwd", inputs, ctx.geo, None, stat, o32, (do, dq, dk, dv, dtable))
        return dq, dk, dv, dtable, None, None, None, None


def _attention(what, q, k, v, heads, kv_heads, scale, mask, q_mask, buckets=None, table=None, offset=0):
    _tensors(what, q, (("k", k), ("v", v), ("mask", mask), ("q_mask", q_mask), ("table", table)))
    heads = int(heads)
    kv_heads = heads if kv_heads is None else int(kv_heads)
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{what}: {heads} heads over {kv_heads} kv heads")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{what}: q, k and v have to be (n, L, heads dk)")
    n, lq, width = q.shape
    if width % heads or not 1 <= width // heads <= MAX_HEAD_DIM:
        raise ValueError(f"{what}: q rows of {width} elements are not {heads} heads of 1 to {MAX_HEAD_DIM}")
    dk = width // heads
    lk = k.shape[1]
    if k.shape != (n, lk, kv_heads * dk) or v.shape != k.shape:
        raise ValueError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} have to be ({n}, Lk, {kv_heads * dk})")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, k and v have to be of one type, float32 or bfloat16")
    for name, m, length in (("mask", mask, lk), ("q_mask", q_mask, lq)):
        if m is not None and (m.dtype != th.bool or m.shape != (n, length)):
            raise ValueError(f"{what}: {name} has to be ({n}, {length}) truth values")
    scale = 1.0 / math.sqrt(dk) if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"{what}: scale {scale} has to be positive")
    lut = None
    if table is not None:
        if not isinstance(buckets, RelativeBuckets):
            raise ValueError(f"{what}: buckets has to be a RelativeBuckets")
        if table.dtype != th.float32 or table.shape != (buckets.n_buckets, heads):
            raise ValueError(f"{what}: table has to be ({buckets.n_buckets}, {heads}) in float32")
        table = table.contiguous()
        lut = buckets.on(q.device)
    inputs = (_rows(q), _rows(k), _rows(v), table, _mask_rows(mask), _mask_rows(q_mask), lut)
    geo = (heads, kv_heads, scale, max(-(1 << 62), min(1 << 62, int(offset))))
    if th.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (table is not None and table.requires_grad)):
        return _Battn.apply(*inputs, geo)
    return _attend(inputs, geo, False)[0]


def cross_attention(q, k, v, heads, kv_heads=None, scale=None, mask=None, q_mask=None):
    """Attention of q's rows over an encoder's states of another length:
    o_i = sum_j softmax_j(scale q_i . k_j) v_j per clip and head, j over the allowed states.

    q (n, Lq, heads dk), k and v (n, Lk, kv_heads dk), float32 or bfloat16, dk <= 128, any strides between
    rows and clips (slices of a joint projection are read in place).  kv_heads divides heads: query head h
    reads kv head h // (heads / kv_heads).  scale: 1 / sqrt(dk) by default, > 0.  mask (n, Lk) / q_mask
    (n, Lq), truth values: the states that may be attended, and the queries that are there; memory of the
    others is not read, their gradients are zero, and so is a row that may attend nothing (or that is
    not there).  Returns (n, Lq, heads dk).  Any lengths from 0 on: few queries over a long memory -- a
    stream's newest frame -- divide the memory among the chip.
    """
    return _attention("cross_attention", q, k, v, heads, kv_heads, scale, mask, q_mask)


def relative_attention(q, k, v, heads, buckets, table, offset=0, kv_heads=None, scale=None, mask=None, q_mask=None):
    """cross_attention with a learned bias by relative position added to the scaled scores:
    s_ij += table[buckets[j - (i + offset)]][head].

    buckets: RelativeBuckets; table (buckets.n_buckets, heads) in float32, with its gradient; an entry of
    -inf forbids its positions.  offset: the position of query row 0 where key row 0 has position 0 -- 0
    over a whole sequence, Lk - Lq for a stream's newest frames over all frames so far.
    """
    if table is None:
        raise ValueError("relative_attention: table has to be a tensor")
    return _attention("relative_attention", q, k, v, heads, kv_heads, scale, mask, q_mask, buckets, table, offset)


# ------------------------------------------------------------------------------------------
# the norms around a block
# ------------------------------------------------------------------------------------------
_KINDS = {"layer": 0, "rms": 1}   # GGD_TR_LAYERNORM, GGD_TR_RMSNORM


def _norm_forward(h, y, gate, weights, geo, keep):
    rows, d, gate_rows, kind, scale, eps = geo
    h_out, u = th.empty_like(h), th.empty_like(h)
    stats = None
    if rows:
        stats = th.empty(4, rows, dtype=th.float32, device=h.device) if keep else None
        _call(native.load().ggd_tr_resnorm_fwd,
              (rows, d, _DTYPES[h.dtype], kind, scale, eps, _p(h), _p(y), _p(gate), gate_rows, *map(_p, weights), _p(h_out), _p(u), _p(stats)),
              h.device, "residual_norm")
    return h_out, u, stats


class _ResidualNorm(th.autograd.Function):
    @staticmethod
    def forward(ctx, h, y, gate, post_g, post_b, pre_g, pre_b, geo):
        h_out, u, stats = _norm_forward(h, y, gate, (post_g, post_b, pre_g, pre_b), geo, True)
        ctx.save_for_backward(h, y, gate, post_g, post_b, pre_g, pre_b, stats)
        ctx.geo = geo
        return h_out, u

    @staticmethod
    @once_differentiable
    def backward(ctx, dh_out, du):
        h, y, gate, post_g, post_b, pre_g, pre_b, stats = ctx.saved_tensors
        rows, d, gate_rows, kind, scale, eps = ctx.geo
        like = lambda t: None if t is None else th.empty_like(t)
        dh, dy, dgate, weights = like(h), like(y), like(gate), [like(w) for w in (post_g, post_b, pre_g, pre_b)]
        if rows == 0:
            return (*(t if t is None else t.zero_() for t in (dh, dy, dgate, *weights)), None)
        dh_out, du = dh_out.contiguous(), du.contiguous()
        lib = native.load()
        nbytes = lib.ggd_tr_resnorm_ws(rows, d, gate_rows, int(gate is not None))
        ws = _workspace(nbytes, h.device)
        _call(lib.ggd_tr_resnorm_bwd,
              (rows, d, _DTYPES[h.dtype], kind, scale, eps, _p(h), _p(y), _p(gate), gate_rows, _p(post_g), _p(post_b), _p(pre_g), _p(pre_b),
               _p(stats), _p(dh_out), _p(du), _p(dh), _p(dy), _p(dgate), *map(_p, weights), _p(ws), nbytes), h.device, "residual_norm backward")
        return (dh, dy, dgate, *weights, None)


def _gate_rows(gate, shape):
    """Rows of h that share a row of the gate, and the gate as it is read: leading dimensions of h, then ones,
    then d; any other shape that broadcasts is expanded."""
    rows = math.prod(shape[:-1])
    if not 1 <= gate.dim() <= len(shape) or any(g not in (1, s) for g, s in zip(gate.shape[::-1], shape[::-1])):
        raise ValueError(f"residual_norm: gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    full = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape)
    at = len(shape) - 1
    while at > 0 and full[at - 1] == 1:
        at -= 1
    if full[-1] != shape[-1] or full[:at] != tuple(shape[:at]):
        return 1, gate.expand(shape).contiguous()
    return max(1, math.prod(shape[at:-1])), gate.contiguous()


def residual_norm(h, y, pre, post=None, gate=None, scale=1.0, kind="layer", eps=1e-5):
    """The step from one block's output to the next block's input in one pass:
    h' = scale h + gate * post(y),  u = pre(h').  Returns (h', u).

    h (the residual stream) and y (the block's output): (..., d) of one shape and type, float32 or bfloat16,
    d <= 8192.  pre and post are (weight, bias) of a norm over d, in float32, bias or the whole of post
    None: LayerNorm (kind "layer") or RMS norm (kind "rms").  gate: of h's type, broadcast to h -- (d,),
    one row a clip (n, 1, d), one a token -- or None.  u is the norm of h' before h' is rounded to its
    type.  Gradients reach h, y, gate and the weights.
    """
    what = "residual_norm"
    for name, pair in (("pre", pre), ("post", post)):
        if not (isinstance(pair, (tuple, list)) and len(pair) == 2 or name == "post" and pair is None):
            raise ValueError(f"{what}: {name} has to be (weight, bias)")
    pre_g, pre_b = pre
    post_g, post_b = (None, None) if post is None else post
    if pre_g is None or (post_g is None and post_b is not None):
        raise ValueError(f"{what}: a norm needs a weight")
    _tensors(what, h, (("y", y), ("gate", gate), ("a weight of pre", pre_g), ("a bias of pre", pre_b), ("a weight of post", post_g),
                       ("a bias of post", post_b)))
    if kind not in _KINDS:
        raise ValueError(f"{what}: kind {kind!r}: layer or rms")
    shape = h.shape
    if h.dim() < 1 or y.shape != shape:
        raise ValueError(f"{what}: h {tuple(shape)} and y {tuple(y.shape)} have to be of one shape")
    if h.dtype not in _DTYPES or y.dtype != h.dtype or (gate is not None and gate.dtype != h.dtype):
        raise ValueError(f"{what}: h, y and gate have to be of one type, float32 or bfloat16")
    d = shape[-1]
    if not 1 <= d <= MAX_NORM_DIM:
        raise ValueError(f"{what}: rows of {d} elements: 1 to {MAX_NORM_DIM}")
    weights = [post_g, post_b, pre_g, pre_b]
    grad = h.requires_grad or y.requires_grad or (gate is not None and gate.requires_grad)
    for i, t in enumerate(weights):
        if t is not None:
            if t.dtype != th.float32 or t.shape != (d,):
                raise ValueError(f"{what}: weights and biases have to be ({d},) in float32")
            grad = grad or t.requires_grad
            weights[i] = t.contiguous()
    scale, eps = float(scale), float(eps)
    if not (math.isfinite(scale) and math.isfinite(eps) and eps > 0):
        raise ValueError(f"{what}: scale {scale} has to be finite, eps {eps} positive")
    gate_rows = 1
    if gate is not None:
        gate_rows, gate = _gate_rows(gate, shape)
    h, y = h.contiguous(), y.contiguous()
    geo = (h.numel() // d, d, gate_rows, _KINDS[kind], scale, eps)
    if grad and th.is_grad_enabled():
        return _ResidualNorm.apply(h, y, gate, *weights, geo)
    return _norm_forward(h, y, gate, weights, geo, False)[:2]
