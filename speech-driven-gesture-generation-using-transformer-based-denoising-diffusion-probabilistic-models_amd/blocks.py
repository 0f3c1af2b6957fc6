"""Operators of a decoder block beyond the reference's: attention for any lengths and padded batches,
attention with a learned relative position bias, and the norms around a block fused with its gate and
residual scale.

They stand beside training.py's operators (linear, layer_norm, squared_relu, ...) and take the same token
matrices, (n, L, heads dk) rows of heads; each is hand-written HIP kernels behind include/ggd_train.h, forward
and backward, in f32 or bf16 with sums, softmax and statistics in f32.  Under torch.no_grad() a call
keeps nothing for a backward pass.  Gradients come once: a second derivative raises.  Everything is issued on the
current stream of the inputs' device, with workspaces from torch's allocator, so that calls on several
streams and captured graphs share nothing; a pass that was run once may be captured.  A captured call with
gradients wants leaves of which no eager graph is alive (a loss kept from before, say), and is refused else.

A wrong shape, type or device raises ValueError before anything is launched.  The checks, the allocations and
the autograd nodes are in csrc/ggd_blocks.cpp.
"""
import operator

import numpy as np
import torch as th

from . import native

MAX_BUCKETS, MAX_DISTANCE = 1024, 2047   # include/ggd_train.h


def _tensor(what, name, t):
    if not isinstance(t, th.Tensor):
        raise ValueError(f"{what}: {name} has to be a tensor")


def _whole(what, name, x):
    """A whole number, of any type that is one (a float is not, whatever its value)."""
    try:
        return operator.index(x)
    except TypeError:
        raise ValueError(f"{what}: {name} {x!r} has to be a whole number") from None


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

    Neither form forbids the keys ahead by itself.  A causal model takes both sides with twice its buckets and a table whose second
    half is -inf: relative_attention(..., torch.cat([table, table.new_full(table.shape, -math.inf)])).
    """

    def __init__(self, n_buckets=32, max_distance=128, both_sides=True, device="cuda"):
        n_buckets, max_distance = _whole("RelativeBuckets", "n_buckets", n_buckets), _whole("RelativeBuckets", "max_distance", max_distance)
        side = n_buckets // 2 if both_sides else n_buckets
        if not 1 <= n_buckets <= MAX_BUCKETS or (both_sides and n_buckets % 2) or side < 2:
            raise ValueError(f"RelativeBuckets: n_buckets {n_buckets}: up to {MAX_BUCKETS}, at least 2 a side, even with both sides")
        if not side // 2 < max_distance <= MAX_DISTANCE:
            raise ValueError(f"RelativeBuckets: max_distance {max_distance}: more than {side // 2}, up to {MAX_DISTANCE}")
        self.n_buckets, self.max_distance, self.both_sides = n_buckets, max_distance, bool(both_sides)
        near, steps = side // 2, side - side // 2
        starts = list(range(near + 1))   # of each bucket of a side; then the least d with d^steps >= near^(steps - k) most^k
        for k in range(1, steps):
            border = near ** (steps - k) * max_distance ** k
            d = round(near * (max_distance / near) ** (k / steps))
            while d ** steps < border:
                d += 1
            while (d - 1) ** steps >= border:
                d -= 1
            starts.append(d)
        of = np.repeat(np.arange(side, dtype=np.int32), np.diff([*starts, max_distance + 1]))   # of |d| = 0 .. max_distance
        ahead = of[1:] + side if both_sides else np.zeros(max_distance, np.int32)
        self.buckets = th.from_numpy(np.concatenate([of[:0:-1], of[:1], ahead]))   # of d = -max_distance .. max_distance
        self._on = {}
        if th.device(device).type != "cpu":
            self.on(th.device(device))

    def __getstate__(self):
        """Without the copies on devices: those of the process that loads it are its own."""
        return dict(self.__dict__, _on={})

    def on(self, device):
        """The buckets on a device, copied there once."""
        device = th.device(device)
        if device.type == "cuda" and device.index is None:
            device = th.device("cuda", th.cuda.current_device())
        if device not in self._on:
            self._on[device] = self.buckets.to(device)
        return self._on[device]


def _attention(what, q, k, v, heads, kv_heads, scale, mask, q_mask, lut, table, offset):
    try:
        return native.load_blocks().attention(what, q, k, v, heads, kv_heads, scale, mask, q_mask, lut, table, offset)
    except TypeError:
        for name, t in (("q", q), ("k", k), ("v", v), ("mask", mask), ("q_mask", q_mask)):
            if t is not None or len(name) == 1:
                _tensor(what, name, t)
        raise ValueError(f"{what}: heads {heads!r} and kv_heads {kv_heads!r} have to be whole numbers, scale {scale!r} a number") from None


def cross_attention(q, k, v, heads, kv_heads=None, scale=None, mask=None, q_mask=None):
    """Attention of q's rows over an encoder's states of another length:
    o_i = sum_j softmax_j(scale q_i . k_j) v_j per clip and head, j over the allowed states.

    q (n, Lq, heads dk), k and v (n, Lk, kv_heads dk), float32 or bfloat16, dk <= 128, any strides between
    rows and clips (slices of a joint projection are read in place).  kv_heads divides heads: query head h
    reads kv head h // (heads / kv_heads).  scale: 1 / sqrt(dk) by default, > 0.  mask (n, Lk) / q_mask
    (n, Lq), truth values: the states that may be attended, and the queries that are there; memory of the
    others is not read, their gradients are zero, and so is a row that may attend nothing (or that is
    not there).  Returns (n, Lq, heads dk).  Lengths from 0 on: few queries over a long memory -- a
    stream's newest frame -- divide the memory among the chip.
    Sums, softmax and statistics are held in f32.  In bfloat16 the weights are rounded once for their product with v (and
    with the gradients) in calls of more than 2^22 scores over more than 64 states, where results are off by that rounding
    and their own; smaller calls, and few queries, carry them to 16 bits, so that the same clip may differ in its last bit alone and
    in a batch.
    (Limits, past which there is a ValueError: 2^28 rows and states; clips x heads x (rows / 32, rounded up) up to 2^22; with
    gradients clips x kv_heads x (states / 128, rounded up) up to 2^22; rows of heads x dk below 32.5 MiB.)
    """
    return _attention("cross_attention", q, k, v, heads, kv_heads, scale, mask, q_mask, None, None, 0)


def relative_attention(q, k, v, heads, buckets, table, offset=0, kv_heads=None, scale=None, mask=None, q_mask=None):
    """cross_attention with a learned bias by relative position added to the scaled scores:
    s_ij += table[buckets[j - (i + offset)]][head].

    buckets: RelativeBuckets; table (buckets.n_buckets, heads) in float32, with its gradient; an entry of
    -inf forbids its positions.  offset: the position of query row 0 where key row 0 has position 0 -- 0
    over a whole sequence, Lk - Lq for a stream's newest frames over all frames so far.
    """
    what = "relative_attention"
    _tensor(what, "table", table)
    if not isinstance(buckets, RelativeBuckets):
        raise ValueError(f"{what}: buckets has to be a RelativeBuckets")
    if table.dtype != th.float32 or table.shape != (buckets.n_buckets, heads):
        raise ValueError(f"{what}: table has to be ({buckets.n_buckets}, {heads}) in float32")
    lut = buckets.on(table.device) if table.is_cuda else None
    return _attention(what, q, k, v, heads, kv_heads, scale, mask, q_mask, lut, table,
                      max(-(1 << 62), min(1 << 62, _whole(what, "offset", offset))))


# ------------------------------------------------------------------------------------------
# the norms around a block
# ------------------------------------------------------------------------------------------
_KINDS = {"layer": 0, "rms": 1}   # GGD_TR_LAYERNORM, GGD_TR_RMSNORM


def residual_norm(h, y, pre, post=None, gate=None, scale=1.0, kind="layer", eps=1e-5):
    """The step from one block's output to the next block's input in one pass:
    h' = scale h + gate * post(y),  u = pre(h').  Returns (h', u).

    h (the residual stream) and y (the block's output): (..., d) of one shape and type, float32 or bfloat16,
    d <= 8192.  pre and post are (weight, bias) of a norm over d, in float32, bias or the whole of post
    None: LayerNorm (kind "layer") or RMS norm (kind "rms").  gate: of h's type, broadcast to h -- (d,),
    one row a clip (n, 1, d), one a token -- or None; another shape that broadcasts (one row a frame, one element a
    token) is expanded to h's, and its gradient summed in f32.  u is the norm of h' before h' is rounded to its
    type.  Gradients reach h, y, gate and the weights.
    """
    what = "residual_norm"
    try:
        pre_g, pre_b = pre
        post_g, post_b = (None, None) if post is None else post
    except (TypeError, ValueError):
        raise ValueError(f"{what}: pre and post have to be (weight, bias)") from None
    if not isinstance(kind, str) or kind not in _KINDS:
        raise ValueError(f"{what}: kind {kind!r}: layer or rms")
    try:
        numbers = float(scale), float(eps)
    except (TypeError, ValueError, OverflowError):
        raise ValueError(f"{what}: scale {scale!r} and eps {eps!r} have to be numbers") from None
    try:
        return native.load_blocks().residual_norm(h, y, pre_g, pre_b, post_g, post_b, gate, numbers[0], _KINDS[kind], numbers[1])
    except TypeError:
        for name, t in (("h", h), ("y", y)):
            _tensor(what, name, t)
        raise ValueError(f"{what}: weights, biases and gate have to be tensors or None") from None
