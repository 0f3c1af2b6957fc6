"""The decoder-block operators on the GPU (…_amd/blocks.py over include/ggd_train.h): cross_attention,
relative_attention and residual_norm against their formulas in 64 bits.

Tolerances are element-wise bounds worked out before the first run from the formulas (attention_bounds,
norm_bounds): a sum of N products in f32 is off by at most N 2^-24 of the sum of their sizes in any
order, a rounding to bf16 by 2^-8 of the value, and both are carried through to each output.
"""
import math

import pytest
import torch as th

pytestmark = pytest.mark.gpu

U = 2.0 ** -24   # half a step of f32
DTYPES = {"f32": th.float32, "bf16": th.bfloat16}
HALF = {"f32": U, "bf16": 2.0 ** -8}   # torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def tr(pkg):
    import importlib
    return importlib.import_module(pkg.__name__ + ".training")


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
def heads_of(x, heads):
    """(n, L, heads dk) -> (n, heads, L, dk) in 64 bits on the CPU."""
    n, length, width = x.shape
    return x.detach().cpu().double().reshape(n, length, heads, width // heads).transpose(1, 2)


def rows_of(x):
    n, heads, length, dk = x.shape
    return x.transpose(1, 2).reshape(n, length, heads * dk)


def attention_formula(q, k, v, do, heads, kv_heads, scale, mask, q_mask, line=None, table=None):
    """Outputs, gradients and their error bounds for f32 sums, each laid out as the operator returns it.
    line: the bucket of every (i, j) as an (lq, lk) tensor."""
    n, lq, lk, dk = q.shape[0], q.shape[1], k.shape[1], q.shape[2] // heads
    group = heads // kv_heads
    Q, dO = heads_of(q, heads), heads_of(do, heads)
    K, V = (heads_of(x, kv_heads).repeat_interleave(group, 1) for x in (k, v))
    allowed = th.ones(n, 1, lq, lk, dtype=th.bool)
    if mask is not None:
        mask = mask.cpu()
        allowed = allowed & mask[:, None, None, :]
        K, V = (x.masked_fill(~mask[:, None, :, None], 0.) for x in (K, V))
    if q_mask is not None:
        q_mask = q_mask.cpu()
        allowed = allowed & q_mask[:, None, :, None]
        Q, dO = (x.masked_fill(~q_mask[:, None, :, None], 0.) for x in (Q, dO))
    s = Q @ K.transpose(-1, -2) * scale
    size = Q.abs() @ K.abs().transpose(-1, -2) * scale   # of the terms of a score
    if table is not None:
        b = table.detach().cpu().double().t()[:, line][None]
        s, size = s + b, size + b.abs().nan_to_num(posinf=0., neginf=0.).clamp(max=1e4)
    s = s.masked_fill(~allowed, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = th.exp(s - m.masked_fill(m == -math.inf, 0.)) * (s > -math.inf)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    o = p @ V
    dV = p.transpose(-1, -2) @ dO
    dp = dO @ V.transpose(-1, -2)
    delta = (dO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # a score is off by dk products and a few roundings; a weight relative by twice that, its sum and exp2
    e_s = ((dk + 6) * U * size).amax(-1, keepdim=True)
    e_p = 2 * e_s + (lk + 16) * U
    half = HALF["f32" if q.dtype == th.float32 else "bf16"]
    e_w = e_p + (half if half > U else 0.)       # bf16: the weight is rounded for the second product
    e_o = (e_w + lk * U) * (p @ V.abs())
    e_dv = ((e_w + lq * group * U) * p).transpose(-1, -2) @ dO.abs()
    e_dp = dk * U * (dO.abs() @ V.abs().transpose(-1, -2))
    e_delta = dk * U * (dO.abs() * o.abs()).sum(-1, keepdim=True) + (dO.abs() * e_o).sum(-1, keepdim=True)
    e_ds = p * (e_p * (dp.abs() + delta.abs()) + e_dp + e_delta + 4 * U * (dp.abs() + delta.abs()))
    e_r = e_ds + (half if half > U else 0.) * (ds.abs() + e_ds)
    e_dq = scale * ((e_r + lk * U * ds.abs()) @ K.abs())
    e_dk = scale * ((e_r + lq * group * U * ds.abs()).transpose(-1, -2) @ Q.abs())
    dQ, dK = scale * ds @ K, scale * ds.transpose(-1, -2) @ Q

    def shared(x):
        return x.reshape(n, kv_heads, group, lk, dk).sum(2)

    out = [rows_of(o), rows_of(dQ), rows_of(shared(dK)), rows_of(shared(dV))]
    err = [rows_of(e_o), rows_of(e_dq), rows_of(shared(e_dk)), rows_of(shared(e_dv))]
    err = [e + half * (x.abs() + e) for e, x in zip(err, out)]
    if table is not None:
        # a wave's 32 rows are added one after another, blocks of 128 rows after each other
        which = th.nn.functional.one_hot(line, table.shape[0]).double()
        out.append(th.einsum("nhij,ijb->bh", ds, which))
        err.append(th.einsum("nhij,ijb->bh", e_ds + n * (lq + lk) * U * ds.abs(), which) + U * out[-1].abs())
    return out, err


def close(got, want, err, what=""):
    got = got.detach().cpu().double()
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    assert bool(th.isfinite(got).all()), what + ": not finite"
    over = ((got - want).abs() - err).max().item() if got.numel() else 0.
    assert over <= 1e-30, (what, over, (got - want).abs().max().item(), err.max().item())


def make_mask(kind, n, length, g):
    if kind == "none":
        return None
    at = th.arange(length)[None]
    keep = at < th.randint(1, length + 1, (n, 1), generator=g)
    if kind == "holes":
        keep = (th.rand(n, length, generator=g) < 0.6)
        keep[-1] = False   # a clip whose mask leaves nothing
    return keep.cuda()


def bucket_line(buckets, lq, lk, offset):
    d = th.arange(lk)[None] - th.arange(lq)[:, None] - offset
    return buckets.buckets.long()[d.clamp(-buckets.max_distance, buckets.max_distance) + buckets.max_distance]


def run_attention(pkg, inputs, do, heads, kv_heads, scale=None, mask=None, q_mask=None, buckets=None, offset=0):
    leaves = [x.detach().clone().requires_grad_() for x in inputs]
    if buckets is None:
        o = pkg.cross_attention(*leaves, heads, kv_heads=kv_heads, scale=scale, mask=mask, q_mask=q_mask)
    else:
        o = pkg.relative_attention(*leaves[:3], heads, buckets, leaves[3], offset=offset, kv_heads=kv_heads, scale=scale,
                                   mask=mask, q_mask=q_mask)
    return [o, *th.autograd.grad(o, leaves, do)]


def check_attention(pkg, inputs, do, heads, kv_heads, mask=None, q_mask=None, buckets=None, offset=0, scale=None):
    q, k, v = inputs[:3]
    dk = q.shape[2] // heads
    got = run_attention(pkg, inputs, do, heads, kv_heads, scale, mask, q_mask, buckets, offset)
    line = None if buckets is None else bucket_line(buckets, q.shape[1], k.shape[1], offset)
    want, err = attention_formula(q, k, v, do, heads, kv_heads, scale or 1 / math.sqrt(dk), mask, q_mask, line,
                                  None if buckets is None else inputs[3])
    for name, a, b, e in zip(("o", "dq", "dk", "dv", "dtable"), got, want, err):
        close(a, b, e, name)
    # the form that keeps nothing gives the same bits
    with th.no_grad():
        if buckets is None:
            o = pkg.cross_attention(q, k, v, heads, kv_heads=kv_heads, scale=scale, mask=mask, q_mask=q_mask)
        else:
            o = pkg.relative_attention(q, k, v, heads, buckets, inputs[3], offset=offset, kv_heads=kv_heads, scale=scale,
                                       mask=mask, q_mask=q_mask)
    assert th.equal(o, got[0])
    return got


def attention_inputs(dtype, n, lq, lk, heads, kv_heads, dk, seed=0, n_buckets=0):
    g = th.Generator().manual_seed(seed)
    shapes = [(n, lq, heads * dk), (n, lk, kv_heads * dk), (n, lk, kv_heads * dk), (n, lq, heads * dk)]
    q, k, v, do = (th.randn(s, generator=g).to(DTYPES[dtype]).cuda() for s in shapes)
    ins = [q, k, v] + ([th.randn(n_buckets, heads, generator=g).cuda()] if n_buckets else [])
    return ins, do, g


# n, lq, lk, heads, kv_heads, dk: one of each; single rows; edges of 32, 64 and 128; heads that fill an image and that
# do not; odd heads; few rows over a memory long enough to be divided, alone and with several tiles of rows
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 33, 4, 2, 32), (3, 40, 32, 8, 8, 32), (2, 65, 129, 4, 1, 64), (1, 130, 70, 2, 2, 128),
          (2, 33, 257, 6, 3, 40), (1, 5, 1000, 2, 1, 80), (2, 7, 2100, 4, 4, 64), (1, 100, 1500, 2, 1, 16), (1, 200, 31, 3, 1, 5),
          (2, 128, 128, 2, 1, 96), (1, 300, 20, 1, 1, 33)]


@pytest.mark.parametrize("mask", ["none", "ragged", "holes"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_cross_attention_and_gradients(pkg, shape, dtype, mask):
    n, lq, lk, heads, kv_heads, dk = shape
    ins, do, g = attention_inputs(dtype, *shape)
    check_attention(pkg, ins, do, heads, kv_heads, mask=make_mask(mask, n, lk, g))


@pytest.mark.parametrize("mask", ["none", "holes"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("plan", [(32, 128, True, 0), (8, 5, True, 3), (6, 20, False, -7), (64, 700, True, 40)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_relative_attention_and_gradients(pkg, shape, dtype, mask, plan):
    n, lq, lk, heads, kv_heads, dk = shape
    buckets = pkg.RelativeBuckets(*plan[:3])
    ins, do, g = attention_inputs(dtype, *shape, n_buckets=plan[0])
    offset = plan[3] if plan[3] else max(0, lk - lq)
    check_attention(pkg, ins, do, heads, kv_heads, mask=make_mask(mask, n, lk, g), buckets=buckets, offset=offset)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk", [(40, 40), (1, 300), (150, 90)])
def test_masked_memory_reaches_nothing(pkg, dtype, lq, lk):
    """NaN, infinities and the type's lowest value where the masks forbid: in q, k, v and in the incoming gradient."""
    n, heads, kv_heads, dk = 3, 4, 2, 32
    buckets = pkg.RelativeBuckets(16, 50)
    ins, do, g = attention_inputs(dtype, n, lq, lk, heads, kv_heads, dk, n_buckets=16)
    mask = make_mask("holes", n, lk, g)
    q_mask = (th.rand(n, lq, generator=g) < 0.7).cuda()
    want = run_attention(pkg, ins, do, heads, kv_heads, None, mask, q_mask, buckets, 2)
    check_attention(pkg, ins, do, heads, kv_heads, mask=mask, q_mask=q_mask, buckets=buckets, offset=2)
    for value in (math.nan, math.inf, -math.inf, th.finfo(DTYPES[dtype]).min):
        bad = [ins[0].masked_fill(~q_mask[..., None], value), ins[1].masked_fill(~mask[..., None], value),
               ins[2].masked_fill(~mask[..., None], value), ins[3]]
        got = run_attention(pkg, bad, do.masked_fill(~q_mask[..., None], value), heads, kv_heads, None, mask, q_mask, buckets, 2)
        for a, b in zip(got, want):
            assert th.equal(a, b)
    assert not want[0][~q_mask].any() and not want[1][~q_mask].any()
    assert not want[0][-1].any() and not want[2][~mask].any() and not want[3][~mask].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk", [(40, 40), (2, 200), (140, 60)])
def test_table_entries_that_forbid_and_that_are_lowest(pkg, dtype, lq, lk):
    """-inf forbids a bucket's places (a row of nothing else is zeros); rows whose every place has the type's lowest value
    are a softmax among equals."""
    n, heads, dk = 2, 2, 32
    buckets = pkg.RelativeBuckets(8, 16)
    ins, do, _ = attention_inputs(dtype, n, lq, lk, heads, heads, dk, n_buckets=8)
    table = ins[3].clone()
    table[2, 0] = -math.inf       # one bucket of head 0
    table[:, 1] = -math.inf       # every bucket of head 1
    got = check_attention(pkg, [*ins[:3], table], do, heads, heads, buckets=buckets)
    assert not got[0][..., dk:].any() and not got[1][..., dk:].any() and not got[4][:, 1].any()
    # among equals: p = 1 / lk whatever the scores, which are lost beside the lowest value
    table = th.full_like(ins[3], th.finfo(th.float32).min)
    q0 = th.zeros_like(ins[0])
    got = run_attention(pkg, [*ins[:3], table], do, heads, heads, buckets=buckets)
    want, err = attention_formula(q0, ins[1], ins[2], do, heads, heads, 1 / math.sqrt(dk), None, None)
    close(got[0], want[0], err[0], "o")
    close(got[3], want[3], err[3], "dv")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dk", [(4, 2, 64), (3, 3, 20)])
def test_strides_slices_and_alignment(pkg, dtype, heads, kv_heads, dk):
    """Slices of joint projections, every second row, expanded clips, and bases that are not 16-byte aligned."""
    n, lq, lk = 2, 50, 70
    g = th.Generator().manual_seed(5)
    wq, wk = heads * dk, kv_heads * dk
    joint = th.randn(n, lk, 2, wq + 2 * wk + 3, generator=g).to(DTYPES[dtype]).cuda()
    one = joint[:, :, 1]
    do = th.randn(n, lq, wq, generator=g).to(DTYPES[dtype]).cuda()
    for shift in (0, 3):
        q, k, v = one[:, :lq, shift:shift + wq], one[..., wq:wq + wk], one[..., wq + wk + shift:wq + 2 * wk + shift]
        for views in ((q, k, v), (q[:1].expand(n, -1, -1), k, v[1:].expand(n, -1, -1)), (q, k.flip(1), v.transpose(1, 2).contiguous().transpose(1, 2))):
            leaves = [x.detach().requires_grad_() for x in views]
            assert all(a.stride() == b.stride() for a, b in zip(leaves, views))
            o = pkg.cross_attention(*leaves, heads, kv_heads=kv_heads)
            got = [o, *th.autograd.grad(o, leaves, do)]
            want, err = attention_formula(*views, do, heads, kv_heads, 1 / math.sqrt(dk), None, None)
            for a, b, e in zip(got, want, err):
                close(a, b, e)
    # a gradient that is itself a view
    wide = th.randn(n, lq, 2 * wq, generator=g).to(DTYPES[dtype]).cuda()
    leaves = [x.detach().requires_grad_() for x in views]
    got = th.autograd.grad(pkg.cross_attention(*leaves, heads, kv_heads=kv_heads), leaves, wide[..., ::2])
    want, err = attention_formula(*views, wide[..., ::2], heads, kv_heads, 1 / math.sqrt(dk), None, None)
    for a, b, e in zip(got, want[1:], err[1:]):
        close(a, b, e)


def test_rows_whose_offsets_pass_32_bits(pkg):
    """Keys and values 2^20 elements apart: the last of 2600 rows lies past 2^31 elements."""
    lk, dk, step = 2600, 64, 1 << 20
    store = th.zeros(lk * step + 2 * dk, dtype=th.bfloat16, device="cuda")
    k, v = store.as_strided((1, lk, dk), (0, step, 1)), store.as_strided((1, lk, dk), (0, step, 1), dk)
    g = th.Generator().manual_seed(6)
    k.copy_(th.randn(1, lk, dk, generator=g)), v.copy_(th.randn(1, lk, dk, generator=g))
    for lq in (1, 700):
        q, do = (th.randn(1, lq, dk, generator=g).bfloat16().cuda() for _ in range(2))
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        o = pkg.cross_attention(*leaves, 1)
        # gradients are laid out anew, without the gaps
        got = [o, *th.autograd.grad(o, leaves, do)]
        want, err = attention_formula(q, k, v, do, 1, 1, 1 / 8, None, None)
        for a, b, e in zip(got, want, err):
            close(a, b, e)
        del leaves, o, got
    del store, k, v
    th.cuda.empty_cache()


def test_large_offsets_and_scales(pkg):
    """Offsets past 32 bits are the table's last buckets; scales other than 1 / sqrt(dk)."""
    ins, do, _ = attention_inputs("f32", 1, 40, 50, 2, 2, 32, n_buckets=8)
    buckets = pkg.RelativeBuckets(8, 16)
    for offset, near in ((1 << 40, 1 << 20), (-(1 << 40), -(1 << 20)), ((1 << 31) + 5, 1 << 20)):
        got = run_attention(pkg, ins, do, 2, 2, buckets=buckets, offset=offset)
        want = run_attention(pkg, ins, do, 2, 2, buckets=buckets, offset=near)
        assert all(th.equal(a, b) for a, b in zip(got, want))
    for scale in (1.0, 0.01):
        check_attention(pkg, ins, do, 2, 2, buckets=buckets, scale=scale)


@pytest.mark.parametrize("n,lq,lk", [(0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0)])
def test_lengths_of_zero(pkg, n, lq, lk):
    buckets = pkg.RelativeBuckets(8, 16)
    ins, do, _ = attention_inputs("bf16", n, lq, lk, 4, 2, 16, n_buckets=8)
    for b in (None, buckets):
        got = run_attention(pkg, ins if b else ins[:3], do, 4, 2, buckets=b)
        assert all(tuple(x.shape) == tuple(y.shape) and not x.any() for x, y in zip(got, [ins[0], *ins]))


@pytest.mark.parametrize("shape", [(2, 300, 500, 4, 2, 64), (1, 3, 3000, 4, 1, 128), (1, 2000, 40, 4, 1, 32)], ids=str)
def test_attention_has_one_order(pkg, shape):
    """The same bits every time, alone and beside other work on a second stream."""
    n, lq, lk, heads, kv_heads, dk = shape
    buckets = pkg.RelativeBuckets(32, 100)
    ins, do, _ = attention_inputs("bf16", *shape, n_buckets=32)
    first = run_attention(pkg, ins, do, heads, kv_heads, buckets=buckets)
    other = th.cuda.Stream()
    other.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(other):
        beside = [run_attention(pkg, ins, do, heads, kv_heads, buckets=buckets) for _ in range(3)]
    again = [run_attention(pkg, ins, do, heads, kv_heads, buckets=buckets) for _ in range(3)]
    th.cuda.synchronize()
    for got in beside + again:
        assert all(th.equal(a, b) for a, b in zip(got, first))


def test_attention_gradients_against_differences(pkg):
    """Central differences of sum(o w) along random directions, in f32: the slope of a step of h is off by h^2 of the third
    derivative (taken as the slope's own size) and by the rounding of two sums over the step."""
    n, lq, lk, heads, kv_heads, dk = 2, 9, 13, 4, 2, 16
    buckets = pkg.RelativeBuckets(8, 12)
    ins, w, g = attention_inputs("f32", n, lq, lk, heads, kv_heads, dk, n_buckets=8)
    mask = make_mask("ragged", n, lk, g)
    grads = run_attention(pkg, ins, w, heads, kv_heads, mask=mask, buckets=buckets)[1:]

    def value(xs):
        with th.no_grad():
            o = pkg.relative_attention(*xs[:3], heads, buckets, xs[3], kv_heads=kv_heads, mask=mask)
        return (o.double() * w.double()).sum().item()

    for at in range(4):
        direction = th.randn(ins[at].shape, generator=g).cuda()
        direction /= direction.norm()
        h = 2.0 ** -5
        slope = (value([x + h * direction if i == at else x for i, x in enumerate(ins)]) -
                 value([x - h * direction if i == at else x for i, x in enumerate(ins)])) / (2 * h)
        size = w.double().abs().sum().item() * 4   # of o: a weighted mean of values below 4
        want = (grads[at].double() * direction.double()).sum().item()
        norm = grads[at].double().norm().item()
        assert abs(slope - want) <= 16 * h * h * norm + 64 * U * size / h, (at, slope, want)


def test_attention_captured_and_replayed(pkg):
    """Forward, and forward with backward, in two graphs that share the allocator's pool; replays in turn with eager work."""
    n, lq, lk, heads, kv_heads, dk = 2, 3, 2000, 4, 2, 64
    buckets = pkg.RelativeBuckets(16, 40)
    ins, do, g = attention_inputs("bf16", n, lq, lk, heads, kv_heads, dk, n_buckets=16)
    fixed = [x.clone().requires_grad_() for x in ins]

    def forward():
        with th.no_grad():
            return pkg.relative_attention(*fixed[:3], heads, buckets, fixed[3], offset=lk - lq, kv_heads=kv_heads)

    def both():
        o = pkg.relative_attention(*fixed[:3], heads, buckets, fixed[3], offset=lk - lq, kv_heads=kv_heads)
        return [o.detach(), *th.autograd.grad(o, fixed, do)]

    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(side):   # no eager graph of these leaves is alive when the capture begins
        forward(), both()
    th.cuda.current_stream().wait_stream(side)
    th.cuda.synchronize()
    g1, g2 = th.cuda.CUDAGraph(), th.cuda.CUDAGraph()
    with th.cuda.graph(g1):
        o1 = forward()
    with th.cuda.graph(g2, pool=g1.pool()):
        o2 = both()
    for step in range(4):
        new, _, _ = attention_inputs("bf16", n, lq, lk, heads, kv_heads, dk, seed=20 + step, n_buckets=16)
        with th.no_grad():
            for a, b in zip(fixed, new):
                a.copy_(b)
        want = run_attention(pkg, new, do, heads, kv_heads, buckets=buckets, offset=lk - lq)
        g1.replay()
        th.cuda.synchronize()
        assert th.equal(o1, want[0])
        g2.replay()
        th.cuda.synchronize()
        assert all(th.equal(a, b) for a, b in zip(o2, want))


def test_a_capture_beside_an_eager_graph_is_refused(pkg):
    """A gradient of the captured pass would draw the eager graph's stream into the capture: refused before, and
    allowed once that graph is gone."""
    x = attention_inputs("f32", 1, 9, 9, 2, 2, 16)[0][0].requires_grad_()
    w = th.ones(32, device="cuda", requires_grad=True)
    with th.no_grad():
        pkg.cross_attention(x, x, x, 2), pkg.residual_norm(x, x, (w, None))

    def attend(t):
        return pkg.cross_attention(t, t, t, 2)

    for call in (lambda: attend(x), lambda: attend(x[:, 1:]), lambda: pkg.residual_norm(x, x.detach(), (w, None))[1],
                 lambda: pkg.residual_norm(x.detach(), x.detach(), (w, None))[1]):
        alive = call()
        with pytest.raises(ValueError, match="eager graph"):
            with th.cuda.graph(th.cuda.CUDAGraph()):
                x.detach() + 1   # (a capture of something)
                call()
        with th.no_grad():   # without gradients there is nothing to refuse
            graph = th.cuda.CUDAGraph()
            with th.cuda.graph(graph):
                o = call()
        graph.replay()
        th.cuda.synchronize()
        assert th.equal(o, alive.detach())
        del alive
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph):
            o = call()
            grads = th.autograd.grad(o, [t for t in (x, w) if o.grad_fn is not None], th.ones_like(o), allow_unused=True)
        graph.replay()
        th.cuda.synchronize()
        want = call()
        assert th.equal(o.detach(), want.detach())
        for a, b in zip(grads, th.autograd.grad(want, [x, w], th.ones_like(want), allow_unused=True)):
            assert (a is None) == (b is None) and (a is None or th.equal(a, b))
        del o, want, grads


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_widest_heads_with_the_longest_distance(pkg, dtype):
    """The largest histograms and images that share the LDS, and the most buckets."""
    buckets = pkg.RelativeBuckets(1024, 2047)
    ins, do, _ = attention_inputs(dtype, 1, 150, 140, 2, 1, 128, n_buckets=1024)
    check_attention(pkg, ins, do, 2, 1, buckets=buckets, offset=-3)


@pytest.mark.parametrize("relative", [False, True])
@pytest.mark.parametrize("lk", [2, 5, 33, 64])
def test_gradients_of_peaked_rows_over_few_keys(pkg, lk, relative):
    """Rows whose weight lies on one key: ds are differences of nearly equal numbers there, and have to come from a delta
    without bf16's roundings.  What is left is half a step (2^-8) of each ds in its product and of the result, and f32's
    share: a score is off by (dk + 8) 2^-23 of the sum of its terms' sizes, exp by some steps, and dp like a score."""
    n, lq, heads, dk = 2, 70, 2, 64
    ins, do, _ = attention_inputs("bf16", n, lq, lk, heads, heads, dk, seed=lk, n_buckets=8 if relative else 0)
    ins[0] = (ins[0] * 4).bfloat16()
    buckets = pkg.RelativeBuckets(8, 16) if relative else None
    got = run_attention(pkg, ins, do, heads, heads, buckets=buckets)
    Q, K, V, dO = (heads_of(x, heads) for x in (*ins[:3], do))
    s, size = Q @ K.transpose(-1, -2) / 8, Q.abs() @ K.abs().transpose(-1, -2) / 8
    if relative:
        b = ins[3].cpu().double().t()[:, bucket_line(buckets, lq, lk, 0)][None]
        s, size = s + b, size + b.abs()
    p, dp = s.softmax(-1), dO @ V.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    off_p = ((dk + 8) * 2.0 ** -23 * size + 2.0 ** -21).amax(-1, keepdim=True)
    off_dp = (dk + 8) * 2.0 ** -23 * (dO.abs() @ V.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    off = 2.0 ** -8 * ds.abs() + p * 2 * (off_dp + off_p * dp.abs().amax(-1, keepdim=True))
    for name, a, want, err in (("dq", got[1], ds @ K / 8, off @ K.abs() / 8),
                               ("dk", got[2], ds.transpose(-1, -2) @ Q / 8, off.transpose(-1, -2) @ Q.abs() / 8)):
        err = 1.01 * err + 2.0 ** -8 * (want.abs() + err)
        close(a, rows_of(want), rows_of(err), name)
    if relative:   # in f32: off without the rounding of ds
        which = th.nn.functional.one_hot(bucket_line(buckets, lq, lk, 0), 8).double()
        off = p * 2 * (off_dp + off_p * dp.abs().amax(-1, keepdim=True)) + n * (lq + lk) * 2.0 ** -24 * ds.abs()
        close(got[4], th.einsum("nhij,ijb->bh", ds, which), th.einsum("nhij,ijb->bh", off, which), "dtable")


def test_attention_leaves_other_memory_alone(pkg):
    """Outputs lie in fresh tensors: inputs stay as they are, and so does what lies around a view's rows."""
    ins, do, g = attention_inputs("bf16", 2, 33, 45, 2, 1, 24)
    store = th.full((2, 60, 48), 7., dtype=th.bfloat16, device="cuda")
    store[:, :45, 12:36] = ins[1]
    before, k = store.clone(), store[:, :45, 12:36]
    run = [x.clone() for x in (ins[0], ins[2], do)]
    leaves = [ins[0].requires_grad_(), k.requires_grad_(), ins[2].requires_grad_()]
    o = pkg.cross_attention(*leaves, 2, kv_heads=1)
    th.autograd.grad(o, leaves, do)
    assert th.equal(store, before) and all(th.equal(a, b) for a, b in zip(run, (ins[0], ins[2], do)))


# ------------------------------------------------------------------------------------------
# residual_norm
# ------------------------------------------------------------------------------------------
def norm_formula(h, y, gate, pre, post, scale, kind, eps, dh_new, du):
    """Outputs, gradients and error bounds in 64 bits over (rows, d); gate already one row a row."""
    half = HALF["f32" if h.dtype == th.float32 else "bf16"]
    d = h.shape[-1]
    w = lambda pair: [None if t is None else t.detach().cpu().double() for t in pair]
    H, Y, G, dN, dU = (None if t is None else t.detach().cpu().double() for t in (h, y, gate, dh_new, du))
    e_sum = (d + 8) * U

    def norm(x, e_x, pair):
        """hat, 1 / sd, the norm, and the errors of hat and of the norm."""
        c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
        e_c = e_x + (e_sum * x.abs().mean(-1, keepdim=True) + e_x.mean(-1, keepdim=True) if kind == "layer" else 0.) + U * x.abs()
        var = (c * c).mean(-1, keepdim=True)
        r = (var + eps).rsqrt()
        e_r = 0.5 * ((2 * c.abs() * e_c + e_c ** 2).mean(-1, keepdim=True) * r ** 2 + 2 * e_sum)   # relative
        hat = c * r
        e_hat = e_c * r + hat.abs() * (e_r + 4 * U)
        weight, bias = w(pair)
        out = hat * weight + (bias if bias is not None else 0.)
        e_out = weight.abs() * e_hat + 2 * U * (hat * weight).abs() + 2 * U * out.abs()
        return hat, r, e_r, out, e_hat, e_out

    def back(dy, e_dy, hat, e_hat, r, e_r, weight):
        gd, e_gd = dy * weight, e_dy * weight.abs() + U * (dy * weight).abs()
        m2 = (gd * hat).mean(-1, keepdim=True)
        e_m2 = (e_gd * hat.abs() + gd.abs() * e_hat + e_sum * (gd * hat).abs()).mean(-1, keepdim=True)
        m1, e_m1 = (gd.mean(-1, keepdim=True), (e_gd + e_sum * gd.abs()).mean(-1, keepdim=True)) if kind == "layer" else (0., 0.)
        t = gd - m1 - hat * m2
        e_t = e_gd + e_m1 + hat.abs() * e_m2 + e_hat * m2.abs() + 4 * U * (gd.abs() + abs(m1) + (hat * m2).abs())
        return t * r, e_t * r + (t * r).abs() * (e_r + 4 * U)

    zero = th.zeros_like(Y)
    n_y, e_n = Y, zero
    if post is not None and post[0] is not None:
        y_hat, y_r, y_er, n_y, y_eh, e_n = norm(Y, zero, post)
    gated, e_g = (n_y, e_n) if G is None else (G * n_y, G.abs() * e_n + U * (G * n_y).abs())
    new = scale * H + gated
    e_new = e_g + 2 * U * ((scale * H).abs() + gated.abs())
    h_hat, h_r, h_er, u, h_eh, e_u = norm(new, e_new, pre)
    out, err = [new, u], [e_new, e_u]
    dx, e_dx = back(dU, zero, h_hat, h_eh, h_r, h_er, w(pre)[0])
    t, e_t = dN + dx, e_dx + 2 * U * (dN.abs() + dx.abs())
    dgate = None if G is None else (t * n_y, e_t * n_y.abs() + t.abs() * e_n + 2 * U * (t * n_y).abs())
    dy, e_dy = (t, e_t) if G is None else (t * G, e_t * G.abs() + U * (t * G).abs())
    rows = h.shape[0]
    col = lambda x, e: (x.sum(0), (e + (rows + 4) * U * x.abs()).sum(0))
    sums = [col(dU * h_hat, dU.abs() * h_eh), col(dU, zero)]
    if post is not None and post[0] is not None:
        sums += [col(dy * y_hat, e_dy * y_hat.abs() + dy.abs() * y_eh), col(dy, e_dy)]
        dy, e_dy = back(dy, e_dy, y_hat, y_eh, y_r, y_er, w(post)[0])
    out += [scale * t, dy]
    err += [abs(scale) * e_t + U * (scale * t).abs(), e_dy]
    err = [e + half * (x.abs() + e) for e, x in zip(err, out)]
    return out, err, dgate, [(x, e + U * x.abs()) for x, e in sums]


def check_norm(pkg, h, y, pre, post, gate, scale, kind, eps=1e-5, seed=0):
    g = th.Generator().manual_seed(100 + seed)
    dh_new, du = (th.randn(h.shape, generator=g).to(h.dtype).cuda() for _ in range(2))
    leaf = lambda t: None if t is None else t.detach().requires_grad_()   # the view itself
    H, Y, G = leaf(h), leaf(y), leaf(gate)
    PRE, POST = [leaf(t) for t in pre], None if post is None else [leaf(t) for t in post]
    out = pkg.residual_norm(H, Y, PRE, post=POST, gate=G, scale=scale, kind=kind, eps=eps)
    leaves = [t for t in (H, Y, G, *PRE, *(POST or ())) if t is not None]
    got = dict(zip([id(t) for t in leaves], th.autograd.grad(out, leaves, (dh_new, du))))
    d = h.shape[-1]
    flat = lambda t: t.reshape(-1, d)
    rows = None if gate is None else flat(gate.expand(h.shape))
    want, err, dgate, sums = norm_formula(flat(h), flat(y), rows, pre, post, scale, kind, eps, flat(dh_new), flat(du))
    for name, a, b, e in zip(("h'", "u", "dh", "dy"), (*out, got[id(H)], got[id(Y)]), want, err):
        close(flat(a), b, e, name)
    if gate is not None:
        x, e = (t.reshape(h.shape).sum_to_size(gate.shape) for t in (dgate[0], dgate[1] + (h.numel() // d + 4) * U * dgate[0].abs()))
        half = HALF["f32" if h.dtype == th.float32 else "bf16"]
        if gate.numel() != h.numel() and gate.dim() == h.dim() and gate.shape[0] == 1 and h.shape[0] > 1 and gate.shape[1] > 1:
            e = e + half * dgate[0].abs().reshape(h.shape).sum_to_size(gate.shape)   # expanded: each row's is rounded before the sum
        close(got[id(G)], x, e + half * (x.abs() + e), "dgate")
    named = zip(("pre weight", "pre bias", "post weight", "post bias"), (*PRE, *(POST or (None, None))), sums + [(None, None)] * 2)
    for name, t, (x, e) in named:
        if t is not None:
            close(got[id(t)], x, e, "d " + name)
    with th.no_grad():
        plain = pkg.residual_norm(h, y, pre, post=post, gate=gate, scale=scale, kind=kind, eps=eps)
    assert all(th.equal(a, b) for a, b in zip(plain, out))
    return [*out, *got.values()]


def norm_inputs(dtype, shape, gate, kind="layer", post=True, seed=0):
    g = th.Generator().manual_seed(seed)
    d, t = shape[-1], DTYPES[dtype]
    rnd = lambda *s, by=1., to=0.: (th.randn(*s, generator=g) * by + to)
    h, y = rnd(*shape).to(t).cuda(), rnd(*shape, by=0.5, to=0.3).to(t).cuda()
    lead = {"none": None, "model": (d,), "clip": (*shape[:-2], 1, d), "token": shape, "frame": (1, *shape[1:])}[gate]
    G = None if lead is None else rnd(*lead, by=0.3, to=0.5).to(t).cuda()
    pair = lambda: (rnd(d, by=0.2, to=1.).cuda(), rnd(d, by=0.2).cuda() if kind == "layer" else None)
    return h, y, pair(), pair() if post else None, G


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,post,gate,scale", [("layer", True, "clip", 1.0), ("layer", False, "none", 0.5), ("rms", True, "token", -2.0),
                                                  ("rms", False, "model", 1.0), ("layer", True, "frame", 0.75), ("layer", True, "none", 0.0)])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 5, 7), (2, 40, 256), (3, 17, 257), (2, 9, 1024), (1, 33, 1000), (2, 3, 2048), (1, 5, 2050),
                                   (1, 4, 4096), (1, 3, 8192), (1, 2, 8191)], ids=str)
def test_residual_norm_and_gradients(pkg, shape, dtype, kind, post, gate, scale):
    h, y, pre, post, G = norm_inputs(dtype, shape, gate, kind, post)
    check_norm(pkg, h, y, pre, post, G, scale, kind)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_residual_norm_over_many_rows(pkg, dtype):
    """More rows than blocks, groups that no segment divides evenly, and one row a group."""
    for shape, gate in (((5, 1501, 64), "clip"), ((3000, 1, 24), "clip"), ((1, 9000, 130), "model"), ((2000, 3, 40), "clip")):
        h, y, pre, post, G = norm_inputs(dtype, shape, gate)
        check_norm(pkg, h, y, pre, post, G, 0.9, "layer")


def test_residual_norm_strides_alignment_and_shapes(pkg):
    g = th.Generator().manual_seed(9)
    wide = th.randn(3, 20, 2, 130, generator=g).cuda()
    _, _, pre, post, _ = norm_inputs("f32", (1, 1, 128), "none")
    h, y = wide[:, :, 0, 1:129], wide[:, :, 1, 2:130]
    check_norm(pkg, h, y, pre, post, wide[:, :1, 0, :128], 1.0, "layer")
    check_norm(pkg, wide[0, 0, 0, :128], wide[0, 0, 1, :128], pre, None, wide[1, 1, 1, :128], 1.0, "layer")   # one row, no batch
    base = th.randn(4 * 64 + 1, generator=g).cuda()[1:].view(4, 64)   # 4 bytes off
    _, _, pre, post, _ = norm_inputs("f32", (1, 1, 64), "none")
    check_norm(pkg, base, base.flip(0), pre, post, None, 1.0, "layer")
    x4 = th.randn(2, 3, 4, 64, generator=g).cuda()
    for lead in ((2, 3, 1, 64), (2, 1, 1, 64), (64,), (1, 64), (2, 3, 4, 64)):
        check_norm(pkg, x4, x4.flip(2), pre, post, th.randn(lead, generator=g).cuda(), 1.0, "layer")


def test_residual_norm_without_rows_and_partly_frozen(pkg):
    _, _, pre, post, _ = norm_inputs("f32", (1, 1, 16), "none")
    h = th.zeros(0, 3, 16, device="cuda", requires_grad=True)
    pre = [t.requires_grad_() for t in pre]
    out = pkg.residual_norm(h, th.zeros_like(h), pre, post=post, gate=th.ones(0, 1, 16, device="cuda"))
    grads = th.autograd.grad([x.sum() for x in out], [h, *pre])
    assert out[0].shape == h.shape and grads[0].shape == h.shape and not grads[1].any() and not grads[2].any()
    # one output used, and only y asked for
    h, y, pre, post, gate = norm_inputs("f32", (2, 5, 16), "clip")
    full = check_norm(pkg, h, y, pre, post, gate, 1.0, "layer")
    y = y.requires_grad_()
    u = pkg.residual_norm(h, y, pre, post=post, gate=gate)[1]
    (dy,) = th.autograd.grad(u.sum(), [y])
    assert dy.shape == y.shape and bool(th.isfinite(dy).all()) and th.equal(u, full[1])


def test_residual_norm_captured_streams_and_order(pkg):
    h, y, pre, post, gate = norm_inputs("bf16", (4, 300, 512), "clip")
    leaves = [t.detach().clone().requires_grad_() for t in (h, y, gate, *pre, *post)]

    def both():
        out = pkg.residual_norm(leaves[0], leaves[1], leaves[3:5], post=leaves[5:7], gate=leaves[2], scale=0.8)
        return [*(o.detach() for o in out), *th.autograd.grad(out, leaves, (y, h))]

    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(side):
        first = both()
    th.cuda.current_stream().wait_stream(side)
    assert all(th.equal(a, b) for a, b in zip(first, both()))
    th.cuda.synchronize()
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        out = both()
    for step in range(3):
        with th.no_grad():
            leaves[1].copy_(y * (step + 1))
        want = [t.clone() for t in both()]
        graph.replay()
        th.cuda.synchronize()
        assert all(th.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------
def test_a_decoder_block_of_them_trains(pkg, tr):
    """Self-attention with a relative bias, cross-attention to padded speech states and the norms between, over the
    training path's linear and squared_relu: outputs and every gradient against autograd in 64 bits of the formulas.
    f32 throughout; each of the ~40 steps is off by some 10^-6 of its size (see the operators' own tests), and
    2e-4 of the largest value leaves two orders for their passage through each other."""
    n, L, Lm, H, d = 3, 40, 53, 8, 256
    dk = d // H
    g = th.Generator().manual_seed(11)
    rnd = lambda *s, by=1.: th.randn(*s, generator=g) * by
    P = {"wqkv": rnd(3 * d, d, by=d ** -0.5), "wo": rnd(d, d, by=d ** -0.5), "wq": rnd(d, d, by=d ** -0.5),
         "wkv": rnd(2 * d, d, by=d ** -0.5), "wo2": rnd(d, d, by=d ** -0.5), "w1": rnd(4 * d, d, by=d ** -0.5),
         "w2": rnd(d, 4 * d, by=(4 * d) ** -0.5), "table": rnd(32, H, by=0.5), "gate": rnd(n, 1, d, by=0.5)}
    for name in ("a", "b", "c", "pa", "pb", "pc"):
        P[name + "w"], P[name + "b"] = rnd(d, by=0.1) + 1, rnd(d, by=0.1)
    x, mem, out_w = rnd(n, L, d), rnd(n, Lm, d), rnd(n, L, d)
    mask = th.arange(Lm)[None] < th.tensor([[53], [20], [1]])
    buckets = pkg.RelativeBuckets(32, 128)
    line = bucket_line(buckets, L, L, 0)

    def block(p, x, mem, mask, lin, self_attn, cross_attn, resnorm, relu2):
        u = resnorm(x, th.zeros_like(x), (p["aw"], p["ab"]), None, None)[1]
        qkv = lin(u, p["wqkv"])
        s = lin(self_attn(qkv[..., :d], qkv[..., d:2 * d], qkv[..., 2 * d:], p["table"]), p["wo"])
        h, u = resnorm(x, s, (p["bw"], p["bb"]), (p["paw"], p["pab"]), p["gate"])
        kv = lin(mem, p["wkv"])
        c = lin(cross_attn(lin(u, p["wq"]), kv[..., :d], kv[..., d:], mask), p["wo2"])
        h, u = resnorm(h, c, (p["cw"], p["cb"]), (p["pbw"], p["pbb"]), p["gate"])
        return resnorm(h, lin(relu2(lin(u, p["w1"])), p["w2"]), (p["pcw"], p["pcb"]), None, p["gate"])[1]

    def ln(v, w, b):
        return (v - v.mean(-1, keepdim=True)) / (v.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b

    def plain_norm(h, y, pre, post, gate):
        y = y if post is None else ln(y, *post)
        h = h + (y if gate is None else gate * y)
        return h, ln(h, *pre)

    def plain_attn(q, k, v, bias=None, mask=None):
        q, k, v = (t.reshape(n, -1, H, dk).transpose(1, 2) for t in (q, k, v))
        s = q @ k.transpose(-1, -2) / math.sqrt(dk)
        if bias is not None:
            s = s + bias.t()[:, line]
        if mask is not None:
            s = s.masked_fill(~mask[:, None, None], -math.inf)
        return (s.softmax(-1) @ v).transpose(1, 2).reshape(n, -1, d)

    def run(dev, dtype, *ops):
        p = {k: v.to(dev, dtype).requires_grad_() for k, v in P.items()}
        X, M = x.to(dev, dtype).requires_grad_(), mem.to(dev, dtype).requires_grad_()
        o = block(p, X, M, mask.to(dev), *ops)
        return [o, *th.autograd.grad(o, [X, M, *p.values()], out_w.to(dev, dtype))]

    got = run("cuda", th.float32, tr.linear, lambda q, k, v, t: pkg.relative_attention(q, k, v, H, buckets, t),
              lambda q, k, v, m: pkg.cross_attention(q, k, v, H, mask=m),
              lambda h, y, pre, post, gate: pkg.residual_norm(h, y, pre, post=post, gate=gate), tr.squared_relu)
    want = run("cpu", th.float64, lambda a, w: a @ w.t(), lambda q, k, v, t: plain_attn(q, k, v, bias=t),
               lambda q, k, v, m: plain_attn(q, k, v, mask=m), plain_norm, lambda a: a.clamp(min=0) ** 2)
    for name, a, b in zip(["out", "x", "mem", *P], got, want):
        err, size = (a.detach().cpu().double() - b).abs().max().item(), b.abs().max().item()
        assert err <= 2e-4 * max(size, 1e-3), (name, err, size)


def test_refusals(pkg):
    """Wrong shapes, types, devices and values: ValueError before anything is launched."""
    z = lambda *s, dtype=th.float32: th.zeros(*s, dtype=dtype, device="cuda")
    q, k = z(2, 3, 64), z(2, 5, 32)
    b, table = pkg.RelativeBuckets(8, 16), z(8, 4)
    cross, rel = pkg.cross_attention, pkg.relative_attention
    keep = th.ones(2, 5, dtype=th.bool, device="cuda")
    assert rel(q, k, k, 4, b, table, kv_heads=2, mask=keep).shape == q.shape
    for call in (lambda: cross(q, k, k, 4), lambda: cross(q, k, k, 4, kv_heads=3), lambda: cross(q, k, k, 0), lambda: cross(q, k, k, 5, kv_heads=1),
                 lambda: cross(q[0], k, k, 4, kv_heads=2), lambda: cross(q, k, k[:, :4], 4, kv_heads=2), lambda: cross(q, k[:1], k[:1], 4, kv_heads=2),
                 lambda: cross(q.bfloat16(), k, k, 4, kv_heads=2), lambda: cross(q.half(), k.half(), k.half(), 4, kv_heads=2),
                 lambda: cross(q, k.cpu(), k, 4, kv_heads=2), lambda: cross(z(1, 2, 130), z(1, 2, 130), z(1, 2, 130), 1),
                 lambda: cross(q, k, k, 4, kv_heads=2, mask=keep.float()), lambda: cross(q, k, k, 4, kv_heads=2, mask=keep[:, :4]),
                 lambda: cross(q, k, k, 4, kv_heads=2, mask=keep.cpu()), lambda: cross(q, k, k, 4, kv_heads=2, q_mask=keep),
                 lambda: cross(q, k, k, 4, kv_heads=2, scale=0.0), lambda: cross(q, k, k, 4, kv_heads=2, scale=1e-60), lambda: cross(q, k, k, 4, kv_heads=2, scale=math.nan),
                 lambda: rel(q, k, k, 4, b, None, kv_heads=2), lambda: rel(q, k, k, 4, None, table, kv_heads=2),
                 lambda: rel(q, k, k, 4, b, table[:7], kv_heads=2), lambda: rel(q, k, k, 4, b, table.double(), kv_heads=2),
                 lambda: rel(q, k, k, 4, b, table.cpu(), kv_heads=2)):
        with pytest.raises(ValueError):
            call()
    h, w = z(2, 3, 16), z(16)
    norm = pkg.residual_norm
    assert len(norm(h, h, (w, None))) == 2
    for call in (lambda: norm(h, h, None), lambda: norm(h, h, (None, w)), lambda: norm(h, h, (w, w), post=(None, w)), lambda: norm(h, h[:1], (w, w)),
                 lambda: norm(h, h.bfloat16(), (w, w)), lambda: norm(h.half(), h.half(), (w, w)), lambda: norm(h, h, (w[:8], w)),
                 lambda: norm(h, h, (w.bfloat16(), w)), lambda: norm(h, h, (w, w), gate=z(3, 1, 16)), lambda: norm(h, h, (w, w), gate=z(16).bfloat16()),
                 lambda: norm(h, h, (w, w), gate=z(1, 2, 3, 16)), lambda: norm(h, h, (w, w), kind="batch"), lambda: norm(h, h, (w, w), eps=0.0),
                 lambda: norm(h, h, (w, w), eps=1e-60), lambda: norm(h, h, (w, w), scale=1e60),
                 lambda: norm(h, h, (w, w), scale=math.inf), lambda: norm(h, h, w), lambda: norm(h, h.cpu(), (w, w)),
                 lambda: norm(z(1, 8193), z(1, 8193), (z(8193), None)), lambda: norm(z(2, 0), z(2, 0), (z(0), None))):
        with pytest.raises(ValueError):
            call()
    # a second derivative
    x = q.clone().requires_grad_()
    (g,) = th.autograd.grad(cross(x, k, k, 4, kv_heads=2).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        th.autograd.grad(g.sum(), [x])


def test_forward_mode_derivatives_are_refused(pkg):
    """... of the inputs, and of the gradients that come into a backward pass (forward over reverse)."""
    fw = th.autograd.forward_ad
    x, w = th.randn(2, 5, 16, device="cuda", requires_grad=True), th.ones(16, device="cuda")
    for call in (lambda t: pkg.cross_attention(t, t, t, 2), lambda t: pkg.residual_norm(t, t, (w, None))[1]):
        with fw.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fw.make_dual(x.detach(), th.ones_like(x)))
            o = call(x)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                th.autograd.grad(o, [x], fw.make_dual(th.ones_like(o), th.ones_like(o)))
            (plain,) = th.autograd.grad(call(x), [x], th.ones_like(o))   # without a tangent all is as before
        (want,) = th.autograd.grad(call(x), [x], th.ones_like(o))
        assert th.equal(plain, want)


def test_tracing_is_refused_and_counting_modes_are_not(pkg):
    """Modes that only look at the operations torch runs leave a call as it is."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        seen = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen += 1
            return func(*args, **(kwargs or {}))

    x, w = th.randn(2, 5, 16, device="cuda"), th.ones(16, device="cuda")
    for call in (lambda t: pkg.cross_attention(t, t, t, 2), lambda t: pkg.residual_norm(t, t, (w, None))[1]):
        want = call(x)
        with pytest.raises(NotImplementedError, match="traced"):
            th.jit.trace(call, (x,))
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call)(x)
        with Count() as mode:
            got = call(x)
        assert mode.seen and th.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk", [(3, 90), (140, 200)])
def test_each_operand_out_of_line_alone(pkg, lq, lk, dtype):
    """Rows one element past an aligned address, or an odd number of elements apart, beside others that are read in place."""
    n, heads, kv_heads, dk = 2, 4, 2, 40
    ins, do, _ = attention_inputs(dtype, n, lq, lk, heads, kv_heads, dk)
    want = run_attention(pkg, ins, do, heads, kv_heads)
    check_attention(pkg, ins, do, heads, kv_heads)

    def off(x):
        store = th.full((n, x.shape[1], x.shape[2] + 3), 9., dtype=x.dtype, device="cuda")
        view = store[..., 1:-2]
        view.copy_(x)
        return view

    for at in range(4):
        xs = [off(x) if i == at else x for i, x in enumerate((*ins, do))]
        leaves = [x.detach().requires_grad_() for x in xs[:3]]
        o = pkg.cross_attention(*leaves, heads, kv_heads=kv_heads)
        grad = xs[3]
        if at == 3:   # a contiguous gradient off its alignment
            grad = th.empty(do.numel() + 1, dtype=do.dtype, device="cuda")[1:].view(do.shape)
            grad.copy_(do)
        for a, b in zip([o, *th.autograd.grad(o, leaves, grad)], want):
            assert th.equal(a, b), at


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,post", [("layer", True), ("rms", False)])
@pytest.mark.parametrize("shape", [(4500, 2, 64), (20000, 2, 64), (9000, 3, 37), (5000, 7, 130), (1100, 2, 1032), (2500, 3, 1029), (4400, 2, 1000)], ids=str)
def test_residual_norm_with_many_gate_rows(pkg, shape, dtype, kind, post):
    """More gate rows than blocks: waves, and past 1024 columns blocks, have whole gate rows, several of them."""
    h, y, pre, post, G = norm_inputs(dtype, shape, "clip", kind, post)
    check_norm(pkg, h, y, pre, post, G, 0.9, kind)


def test_residual_norm_with_millions_of_gate_rows(pkg):
    """2^22 + 3 gate rows of 2 rows: what belongs to a row or gate row has the bits of the two halves' calls, whose gradients of the
    weights add up (to n U of the sums of sizes)."""
    n, d = (1 << 22) + 3, 8
    g = th.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: th.randn(*s, generator=g, device="cuda")
    h, y, gate, dh, du = rnd(n, 2, d), rnd(n, 2, d), rnd(n, 1, d), rnd(n, 2, d), rnd(n, 2, d)
    w = [1 + 0.1 * rnd(d) for _ in range(4)]

    def call(at):
        leaves = [t.detach().requires_grad_() for t in (h[at], y[at], gate[at], *w)]
        out = pkg.residual_norm(leaves[0], leaves[1], leaves[3:5], post=leaves[5:7], gate=leaves[2], scale=0.5)
        return [o.detach() for o in out] + list(th.autograd.grad(out, leaves, (dh[at], du[at])))

    whole, one, two = call(slice(None)), call(slice(0, n // 2)), call(slice(n // 2, n))
    for a, b, c in zip(whole[:5], one, two):
        assert th.equal(a, th.cat([b, c]))
    # a block adds at most 2 (n / 1024 / 4 + 1) rows a wave one after another, 4 waves, then 2048 / 16 blocks and 16 lists; each term is
    # below 8 * 8 * 3 (a gradient of 8, a norm of sqrt(8) < 3 and a gate below 8, twice over)
    steps = 2 * (n // 4096 + 1) + 4 + 2048 // 16 + 16
    for a, b, c in zip(whole[5:], one[5:], two[5:]):
        assert bool(((a - (b + c)).abs() <= 2 * steps * U * 2 * n * 8).all())


# gates that share elements of other axes than whole trailing rows: one a frame, one a token or clip, one for all, a middle axis
GATES = [((3, 40, 96), (1, 40, 96)), ((3, 40, 96), (40, 96)), ((6, 50, 256), (6, 50, 1)), ((2, 9, 1024), (2, 1, 1)), ((2, 300, 65), (1, 1, 1)),
         ((2, 300, 65), (1,)), ((2, 5, 4, 48), (2, 1, 4, 48)), ((2, 5, 4, 48), (1, 5, 1, 48)), ((2, 3, 5, 4, 8), (1, 3, 1, 4, 1)), ((700, 24), (700, 1)),
         ((1, 5000, 33), (1, 5000, 1)), ((900, 2, 40), (1, 2, 40)), ((7,), (1,))]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape,lead", GATES, ids=str)
def test_gradients_of_gates_that_broadcast_otherwise(pkg, shape, lead, dtype):
    """The gradient of an element is one sum in f32, rounded once."""
    h, y, pre, post, _ = norm_inputs(dtype, (1, *shape) if len(shape) < 2 else shape, "none")
    h, y = h.reshape(shape), y.reshape(shape)
    g = th.Generator().manual_seed(4)
    gate = (th.randn(lead, generator=g) * 0.3 + 0.5).to(h.dtype).cuda()
    dh, du = (th.randn(shape, generator=g).to(h.dtype).cuda() for _ in range(2))
    leaves = [t.detach().requires_grad_() for t in (h, y, gate, *pre, *post)]
    out = pkg.residual_norm(leaves[0], leaves[1], leaves[3:5], post=leaves[5:7], gate=leaves[2], scale=0.7)
    got = th.autograd.grad(out, leaves, (dh, du))
    d = shape[-1]
    flat = lambda t: t.reshape(-1, d)
    want, err, dgate, sums = norm_formula(flat(h), flat(y), flat(gate.expand(shape)), pre, post, 0.7, "layer", 1e-5, flat(dh), flat(du))
    for name, a, b, e in zip(("h'", "u", "dh", "dy"), (*out, *got[:2]), want, err):
        close(flat(a), b, e, name)
    of = h.numel() // gate.numel()
    x, e = (t.reshape(shape).sum_to_size(gate.shape) for t in (dgate[0], dgate[1] + of * U * dgate[0].abs()))
    close(got[2], x, e + HALF[dtype] * (x.abs() + e), "dgate")
    for a, (x, e) in zip(got[3:], sums):
        close(a, x, e)


def test_gates_that_broadcast_otherwise_are_captured(pkg):
    """Replays of a pass whose gates' gradients are sums over other axes, in turn with eager work."""
    g = th.Generator().manual_seed(8)
    rnd = lambda *s: th.randn(*s, generator=g).bfloat16().cuda()
    h, y, dh, du = (rnd(16, 512, 256) for _ in range(4))
    w = th.ones(256, device="cuda")
    for lead in ((1, 512, 256), (16, 512, 1), (1, 1, 1)):
        leaves = [t.clone().requires_grad_() for t in (h, y, rnd(*lead))]

        def both():
            out = pkg.residual_norm(leaves[0], leaves[1], (w, None), gate=leaves[2], kind="rms")
            return [*(o.detach() for o in out), *th.autograd.grad(out, leaves, (dh, du))]

        side = th.cuda.Stream()
        side.wait_stream(th.cuda.current_stream())
        with th.cuda.stream(side):
            both()
        th.cuda.current_stream().wait_stream(side)
        th.cuda.synchronize()
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph):
            out = both()
        for step in range(5):
            with th.no_grad():
                leaves[1].copy_(rnd(16, 512, 256))
            want = [t.clone() for t in both()]
            graph.replay()
            th.cuda.synchronize()
            assert all(th.equal(a, b) for a, b in zip(out, want)), (lead, step)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_that_are_not_asked_for(pkg, dtype):
    """Any operand frozen: the others' gradients have the same bits, and a frozen memory's dk and dv are not formed."""
    n, lq, lk, heads, kv_heads, dk = 2, 70, 1500, 4, 2, 64
    ins, do, _ = attention_inputs(dtype, n, lq, lk, heads, kv_heads, dk, n_buckets=8)
    buckets = pkg.RelativeBuckets(8, 16)
    want = run_attention(pkg, ins, do, heads, kv_heads, buckets=buckets)[1:]
    for wanted in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (0, 1), (2, 3)):
        leaves = [x.detach().requires_grad_(i in wanted) for i, x in enumerate(ins)]
        o = pkg.relative_attention(*leaves[:3], heads, buckets, leaves[3], kv_heads=kv_heads)
        got = th.autograd.grad(o, [leaves[i] for i in wanted], do)
        assert all(th.equal(a, want[i]) for a, i in zip(got, wanted)), wanted
    # dk and dv of a long memory alone would be twice its keys
    q, k = (th.randn(1, rows, 64, device="cuda").to(DTYPES[dtype]) for rows in (8, 1 << 16))
    q.requires_grad_()
    o = pkg.cross_attention(q, k, k, 1)
    before = th.cuda.memory_allocated()
    th.cuda.reset_peak_memory_stats()
    th.autograd.grad(o, [q], th.ones_like(o))
    assert th.cuda.max_memory_allocated() - before < k.numel() * k.element_size()
    h, y, pre, post, _ = norm_inputs(dtype, (3, 20, 64), "none")
    gate = ins[3][:1, :1].to(h.dtype).reshape(1, 1, 1).expand(3, 20, 1).contiguous()
    every = [h, y, gate, *pre, *post]
    call = lambda t: pkg.residual_norm(t[0], t[1], t[3:5], post=t[5:7], gate=t[2])[1]
    leaves = [t.detach().requires_grad_() for t in every]
    want = th.autograd.grad(call(leaves), leaves, h)
    for at in range(7):
        leaves = [t.detach().requires_grad_(i == at) for i, t in enumerate(every)]
        (got,) = th.autograd.grad(call(leaves), [leaves[at]], h)
        assert th.equal(got, want[at]), at


def test_a_plan_let_go_while_another_stream_uses_it(pkg):
    """A plan made on one stream, used on a busy second one and dropped: its memory is not handed on before that use is over."""
    ins, do, _ = attention_inputs("f32", 2, 40, 50, 2, 2, 32, n_buckets=8)
    want = run_attention(pkg, ins, do, 2, 2, buckets=pkg.RelativeBuckets(8, 16))
    busy = th.randn(4096, 4096, device="cuda")
    side = th.cuda.Stream()
    for _ in range(3):
        plan = pkg.RelativeBuckets(8, 16)
        size, at = plan.on("cuda").numel(), plan.on("cuda").data_ptr()
        side.wait_stream(th.cuda.current_stream())
        with th.cuda.stream(side):
            for _ in range(20):
                th.mm(busy, busy)
            got = run_attention(pkg, ins, do, 2, 2, buckets=plan)
        del plan
        others = [th.full((size,), 7, dtype=th.int32, device="cuda") for _ in range(64)]   # on the first stream, at once
        assert all(t.data_ptr() != at for t in others) or side.query()
        th.cuda.synchronize()
        assert all(th.equal(a, b) for a, b in zip(got, want))
        del others


def test_values_negated_when_read(pkg):
    """The imaginary part of a conjugate is a view whose values torch negates when it reads them."""
    g = th.Generator().manual_seed(12)
    neg = lambda *s: th.randn(*s, dtype=th.complex64, generator=g).cuda().conj().imag
    q, k, v = neg(2, 3, 1), neg(2, 5, 1), neg(2, 5, 1)   # one head of one element: rows in place whatever the last stride
    assert q.is_neg() and k.is_neg()
    plain = [x.clone().resolve_neg() for x in (q, k, v)]
    assert not plain[0].is_neg() and th.equal(pkg.cross_attention(q, k, v, 1), pkg.cross_attention(*plain, 1))
    h, y, w, gate = neg(1, 1), neg(1, 1), neg(1), neg(1)
    call = lambda f: pkg.residual_norm(f(h), f(y), (f(w), f(w)), post=(f(w), f(w)), gate=f(gate), kind="rms")
    assert all(th.equal(a, b) for a, b in zip(call(lambda t: t), call(lambda t: t.clone().resolve_neg())))


def test_sparse_tensors_are_refused(pkg):
    x, w = th.ones(2, 3, 16, device="cuda"), th.ones(16, device="cuda")
    keep = th.ones(2, 3, dtype=th.bool, device="cuda")
    buckets, table = pkg.RelativeBuckets(8, 16), th.ones(8, 2, device="cuda")
    for call in (lambda: pkg.cross_attention(x.to_sparse(), x, x, 2), lambda: pkg.cross_attention(x, x, x.to_sparse(), 2),
                 lambda: pkg.cross_attention(x, x, x, 2, mask=keep.to_sparse()), lambda: pkg.relative_attention(x, x, x, 2, buckets, table.to_sparse()),
                 lambda: pkg.residual_norm(x.to_sparse(), x, (w, w)), lambda: pkg.residual_norm(x, x.to_sparse(), (w, w)),
                 lambda: pkg.residual_norm(x, x, (w.to_sparse(), w)), lambda: pkg.residual_norm(x, x, (w, w), gate=w.to_sparse())):
        with pytest.raises(ValueError, match="dense"):
            call()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk,offset", [(70, 70, 0), (300, 300, 0), (1, 90, 89), (5, 200, 195)])
def test_a_causal_table(pkg, lq, lk, offset, dtype):
    """Twice the buckets, the second half's entries -inf: each query attends the keys at and behind it, with the biases of a one-sided
    plan, and the gradients of the learned half are those of the formula."""
    n, heads, kv_heads, dk, s = 2, 4, 2, 32, 12
    both, one = pkg.RelativeBuckets(2 * s, 40), pkg.RelativeBuckets(s, 40, both_sides=False)
    assert th.equal(both.buckets[:41], one.buckets[:41])
    ins, do, _ = attention_inputs(dtype, n, lq, lk, heads, kv_heads, dk, n_buckets=s)
    table = th.cat([ins[3], th.full_like(ins[3], -math.inf)])
    got = check_attention(pkg, [*ins[:3], table], do, heads, kv_heads, buckets=both, offset=offset)
    assert not got[4][s:].any()
    # keys ahead reach nothing, whatever they hold
    if lq == 70:
        late = [x.clone() for x in ins[:3]]
        late[1][:, 40:], late[2][:, 40:] = 3., -5.
        again = run_attention(pkg, [*late, table], do, heads, kv_heads, buckets=both, offset=offset)
        assert th.equal(again[0][:, :40], got[0][:, :40])


def test_a_saved_plan_loaded_elsewhere(pkg, tmp_path):
    ins, do, _ = attention_inputs("f32", 1, 40, 50, 2, 2, 32, n_buckets=8)
    plan = pkg.RelativeBuckets(8, 16)
    want = run_attention(pkg, ins, do, 2, 2, buckets=plan)
    th.save(plan, tmp_path / "plan.pt")
    loaded = th.load(tmp_path / "plan.pt", map_location="cpu", weights_only=False)
    assert all(th.equal(a, b) for a, b in zip(run_attention(pkg, ins, do, 2, 2, buckets=loaded), want))
    plan._on[th.device("cuda", 0)] = plan.buckets   # on the host: refused
    with pytest.raises(ValueError, match="the plan"):
        pkg.relative_attention(*ins[:3], 2, plan, ins[3])


def test_saved_tensors_through_hooks(pkg):
    """Kept on the host in between, or laid out anew: the same gradients.  Come back on the host, of another type or shape: an error."""
    hooks = th.autograd.graph
    ins, do, g = attention_inputs("bf16", 2, 40, 50, 4, 2, 32, n_buckets=8)
    buckets, mask = pkg.RelativeBuckets(8, 16), make_mask("ragged", 2, 50, g)
    joint = th.cat([ins[1], ins[2]], -1)
    h, y, pre, post, _ = norm_inputs("f32", (2, 5, 16), "none")
    gate = th.rand(2, 5, 1, device="cuda")

    def attend():
        leaves = [x.detach().requires_grad_() for x in (ins[0], joint, ins[3])]
        o = pkg.relative_attention(leaves[0], leaves[1][..., :64], leaves[1][..., 64:], 4, buckets, leaves[2], kv_heads=2, mask=mask)
        return o, leaves, do

    def norm():
        leaves = [x.detach().requires_grad_() for x in (h, y, gate, *pre, *post)]
        return pkg.residual_norm(leaves[0], leaves[1], leaves[3:5], post=leaves[5:], gate=leaves[2])[1], leaves, y

    for make in (attend, norm):
        want = th.autograd.grad(*make())
        with hooks.save_on_cpu():
            o = make()
        assert all(th.equal(a, b) for a, b in zip(th.autograd.grad(*o), want))
        with hooks.saved_tensors_hooks(lambda t: t, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)):
            o = make()
        assert all(th.equal(a, b) for a, b in zip(th.autograd.grad(*o), want))
        for spoil in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t.flatten()[:-1], lambda t: t.unsqueeze(0), lambda t: t[..., :1]):
            with hooks.saved_tensors_hooks(lambda t: t, spoil):
                o = make()
            with pytest.raises(RuntimeError, match="saved tensor"):
                th.autograd.grad(*o)


def test_threads_at_once(pkg):
    """Each on a stream of its own, forward and backward: the bits of one alone."""
    import threading
    ins, do, _ = attention_inputs("bf16", 2, 60, 700, 4, 2, 64, n_buckets=8)
    buckets = pkg.RelativeBuckets(8, 16)
    h, y, pre, post, gate = norm_inputs("bf16", (4, 50, 256), "clip")

    def both():
        got = run_attention(pkg, ins, do, 4, 2, buckets=buckets)
        leaves = [t.detach().requires_grad_() for t in (h, y, gate, *pre, *post)]
        out = pkg.residual_norm(leaves[0], leaves[1], leaves[3:5], post=leaves[5:], gate=leaves[2])
        return [*got, *out, *th.autograd.grad(out, leaves, (y, h))]

    want, wrong = both(), []
    th.cuda.synchronize()

    def work():
        stream = th.cuda.Stream()
        with th.cuda.stream(stream):
            for _ in range(20):
                got = both()
                stream.synchronize()
                if not all(th.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_gate_whose_rows_are_not_in_order(pkg):
    """A gate that is a transposed view, of the kinds that are read in place and that are expanded: gradients in its own order."""
    h, y, pre, post, _ = norm_inputs("f32", (3, 20, 64), "none")
    g = th.Generator().manual_seed(5)
    for shape in ((1, 3, 64), (20, 3, 1), (64, 20, 1)):
        base = th.randn(shape, generator=g).cuda()
        views = {(1, 3, 64): lambda t: t.transpose(0, 1), (20, 3, 1): lambda t: t.transpose(0, 1), (64, 20, 1): lambda t: t.permute(2, 1, 0)}
        view = views[shape]
        grads = []
        for leaf in (base.clone().requires_grad_(), view(base).contiguous().requires_grad_()):
            gate = view(leaf) if leaf.shape == base.shape and not grads else leaf
            out = pkg.residual_norm(h, y, pre, post=post, gate=gate)
            (d,) = th.autograd.grad(out, [leaf], (y, h))
            grads.append(view(d) if not grads else d)
        assert th.equal(*grads), shape
        check_norm(pkg, h, y, pre, post, view(base), 1.0, "layer") if shape[-1] == 64 else None
