"""The decoder-block operators' attention in calls of the size that a long training step has: bf16 products rounded once (past 2^22 scores
and 64 keys), keys divided among blocks of 128 rows, dk and dv of wide heads shared by two waves with divided and with long query
axes, and clips' kv heads that do not fill the XCDs in turn.  Formulas and bounds are test_gpu_blocks.py's."""
import math

import pytest
import torch as th

from tests.test_gpu_blocks import U, attention_inputs, bucket_line, check_attention, make_mask, run_attention

pytestmark = pytest.mark.gpu


def masks(n, lq, lk, g):
    """Ragged keys, and queries of which a third is not there."""
    return make_mask("ragged", n, lk, g), (th.rand(n, lq, generator=g) < 0.67).cuda()


# 2 x 8 x 777 x 777 scores are past 2^22; dk and dv: 28 blocks whose 52 tiles of queries are divided, or 112 of 13; the last two have
# 256 blocks with 11 tiles of queries each, undivided
@pytest.mark.parametrize("relative", [False, True])
@pytest.mark.parametrize("shape", [(2, 777, 777, 8, 2, 64), (2, 777, 777, 8, 8, 64), (2, 777, 777, 8, 2, 128), (2, 777, 777, 8, 8, 100),
                                   (8, 700, 500, 8, 8, 128), (8, 700, 500, 8, 8, 32)], ids=str)
def test_bf16_products_rounded_once(pkg, shape, relative):
    n, lq, lk, heads, kv_heads, dk = shape
    assert n * heads * lq * lk > 1 << 22 and lk > 64
    buckets = pkg.RelativeBuckets(20, 200) if relative else None
    ins, do, g = attention_inputs("bf16", *shape, n_buckets=20 if relative else 0)
    mask, q_mask = masks(n, lq, lk, g)
    check_attention(pkg, ins, do, heads, kv_heads, mask=mask, q_mask=q_mask, buckets=buckets)


def test_a_causal_table_in_a_large_call(pkg):
    """The second half of both sides' buckets forbidden: most blocks of keys ahead have no place that is allowed."""
    n, lq, lk, heads, kv_heads, dk = 2, 777, 777, 8, 2, 64
    buckets = pkg.RelativeBuckets(24, 100)
    ins, do, g = attention_inputs("bf16", n, lq, lk, heads, kv_heads, dk, n_buckets=12)
    table = th.cat([ins[3], th.full_like(ins[3], -math.inf)])
    got = check_attention(pkg, [*ins[:3], table], do, heads, kv_heads, mask=make_mask("ragged", n, lk, g), buckets=buckets)
    assert not got[4][12:].any()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,heads,kv_heads,dk", [(8, 8, 8, 64), (8, 8, 2, 128), (16, 4, 1, 32)])
def test_table_gradient_without_the_weights_rounding(pkg, n, heads, kv_heads, dk, masked):
    """The table's gradient is a sum in f32 and has f32's error, though o -- and delta = do . o with it -- comes from rounded weights.

    Keys of even places score 0, those of odd ones ln w with w = (1 + 0.9 2^-8) / 2, which rounds down to 1 / 2; their v . do are
    +1 and -1.  So every row's delta is off to the same side, by (1/2 / (3/2)) - (1 - w) / (1 + w) = 1.6e-3, which sums to
    1.6e-3 p over a bucket's places unless it is taken out.  The bound: a score is off by (dk + 6) U of its terms, a weight by twice that and
    (lk + 16) U, dp by dk U, and the row's mean of dp by its weights' and terms' errors and lk U a sum.  Places are added in f32 within
    a block of 128 rows -- a lane's up to lk, 256 threads' in trees, then up to 2 D + 1 distances, so lk + 2 D + 128 one after
    another at most -- and the blocks in 64 bits; what is taken out is added the same way."""
    lq, lk, D = 420, 200, 24
    assert n * heads * lq * lk > 1 << 22
    buckets = pkg.RelativeBuckets(8, D)
    w = 0.5 * (1 + 0.9 * 2.0 ** -8)
    scale = -math.log(w)
    zero = lambda rows, h: th.zeros(n, rows, h, dk)
    q, k, v, do = zero(lq, heads), zero(lk, kv_heads), zero(lk, kv_heads), zero(lq, heads)
    odd = (th.arange(lk) % 2).float()[None, :, None]
    q[..., 0], k[..., 0], v[..., 0] = 1., -odd, 1 - 2 * odd
    do[..., 0] = 1 + th.arange(heads)[None, None] % 2
    flat = [t.reshape(n, t.shape[1], -1).bfloat16().cuda() for t in (q, k, v, do)]
    g = th.Generator().manual_seed(3)
    mask, q_mask = masks(n, lq, lk, g) if masked else (None, None)
    got = run_attention(pkg, [*flat[:3], th.zeros(8, heads, device="cuda")], flat[3], heads, kv_heads, scale, mask, q_mask, buckets)[4]

    # the formula: one head's places, do scaled by head
    keep = th.ones(n, lk, dtype=th.bool) if mask is None else mask.cpu()
    there = th.ones(n, lq, dtype=th.bool) if q_mask is None else q_mask.cpu()
    at = (th.arange(lk) % 2).double()
    s = -at * float(th.tensor(scale))   # (the kernels' scale is the f32 of it: off by U, within a score's bound)
    p = th.exp(s)[None] * keep
    p = (p / p.sum(-1, keepdim=True))[:, None] * there[..., None]   # (n, lq, lk)
    dp = (1 - 2 * at)[None, None].expand_as(p)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_p = 2 * (dk + 6) * U * scale + (lk + 16) * U
    e_dp = dk * U
    e_mean = (p * ((e_p + (lk + 4) * U) * dp.abs() + e_dp)).sum(-1, keepdim=True) + 2 * lk * U * (delta.abs() + 2.0 ** -8)
    taken = p * 2.0 ** -8   # delta's error is below 2^-8 (a mean of weights' relative errors below that, over |dp| = 1)
    e = p * (e_p * (dp.abs() + delta.abs()) + e_dp + e_mean) + (lk + 2 * D + 128) * U * (ds.abs() + 2 * taken)
    which = th.nn.functional.one_hot(bucket_line(buckets, lq, lk, 0), 8).double()
    per = lambda x: th.einsum("nij,ijb->b", x, which)
    by_head = (1 + th.arange(heads) % 2).double()
    want, err = per(ds)[:, None] * by_head, 1.01 * per(e)[:, None] * by_head
    err = err + U * want.abs()
    missed = per(p * there[..., None])[:, None] * by_head * 1.5e-3   # what would be left without the correction
    assert bool((missed[[3, 7]] > 8 * err[[3, 7]]).all())   # ... in the buckets of most places: far over the bound
    over = ((got.cpu().double() - want).abs() - err).max().item()
    assert over <= 0, (over, (got.cpu().double() - want).abs().max().item(), err.max().item())


@pytest.mark.parametrize("relative", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 300, 700, 4, 2, 64), (1, 200, 700, 4, 4, 128), (2, 140, 500, 3, 3, 33)], ids=str)
def test_many_rows_over_divided_keys(pkg, shape, dtype, relative):
    """Few blocks of 128 rows: the keys divided among blocks, in the forward pass (joined by maxima and sums) and in dq's."""
    n, lq, lk, heads, kv_heads, dk = shape
    buckets = pkg.RelativeBuckets(12, 90) if relative else None
    ins, do, g = attention_inputs(dtype, *shape, n_buckets=12 if relative else 0)
    mask, q_mask = masks(n, lq, lk, g)
    check_attention(pkg, ins, do, heads, kv_heads, mask=mask, q_mask=q_mask, buckets=buckets, offset=lk - lq if relative else 0)
    check_attention(pkg, ins, do, heads, kv_heads, buckets=buckets)


# scores on both sides of 2^24, and of 2^22 for f32 heads past 64: the few rows' kernel gives way to blocks of 128 rows
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 800, 5200, 4, 2, 64), (1, 850, 5200, 4, 2, 64), (2, 140, 3700, 4, 4, 128), (2, 140, 3800, 4, 4, 128)], ids=str)
def test_many_rows_over_far_more_keys(pkg, shape, dtype):
    n, lq, lk, heads, kv_heads, dk = shape
    assert lk >= 4 * lq and n * heads * ((lq + 127) // 128) < 128
    ins, do, g = attention_inputs(dtype, *shape)
    mask, q_mask = masks(n, lq, lk, g)
    check_attention(pkg, ins, do, heads, kv_heads, mask=mask, q_mask=q_mask)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lq,lk", [(1, 40), (40, 33), (130, 70)])
def test_kv_heads_that_do_not_fill_the_xcds(pkg, lq, lk, dtype):
    """66 clips' kv heads, dealt to 8 XCDs in turn: the last round has two."""
    ins, do, g = attention_inputs(dtype, 11, lq, lk, 12, 6, 32)
    check_attention(pkg, ins, do, 12, 6, mask=make_mask("holes", 11, lk, g))


def test_many_heads_over_a_long_memory(pkg):
    """512 heads on 16 kv heads over 270000 states.  Values grow along the memory, so that a part of it left out, or read twice, shows.
    f32: a lane adds every eighth key of one of at least 32 parts one after another, 1055 at most, the parts follow: 1200 U
    of o's terms twice (weights and their sum), and a weight's own error is 2 (dk + 8) U of its score's terms."""
    heads, kv_heads, dk, lk = 512, 16, 8, 270000
    assert heads * (lk // 32) > 1 << 22
    g = th.Generator(device="cuda").manual_seed(1)
    q, k = (th.randn(1, length, h * dk, generator=g, device="cuda") for length, h in ((1, heads), (lk, kv_heads)))
    v = th.linspace(0, 1, lk, device="cuda")[None, :, None] + th.rand(1, lk, kv_heads * dk, generator=g, device="cuda")
    with th.no_grad():
        got = pkg.cross_attention(q, k, v, heads, kv_heads=kv_heads)
    split = lambda x, h: x.double().reshape(-1, h, dk).transpose(0, 1).contiguous()
    Q, K, V = split(q, heads).reshape(kv_heads, heads // kv_heads, dk), split(k, kv_heads), split(v, kv_heads)
    for h in range(kv_heads):
        s, size = Q[h] @ K[h].t() / math.sqrt(dk), Q[h].abs() @ K[h].abs().t() / math.sqrt(dk)
        p = s.softmax(-1)
        want = p @ V[h]
        err = (2 * 1200 * U + 2 * (dk + 8) * U * size.amax(-1, keepdim=True)) * want + U * want
        out = got.reshape(kv_heads, heads // kv_heads, dk)[h].double()
        assert bool(((out - want).abs() <= err).all()), (h, (out - want).abs().max().item(), err.max().item())


@pytest.mark.parametrize("dk", [8, 128])
def test_as_many_heads_as_there_may_be(pkg, dk):
    """2^22 clips' heads of one row over one key: o is v, dv is do, and dq and dk nothing but the rounding of dk products twice."""
    n, heads = 1 << 17, 32
    q, k, v, do = (th.randn(n, 1, heads * dk, device="cuda", dtype=th.bfloat16) for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = pkg.cross_attention(*leaves, heads)
    dq, dk_, dv = th.autograd.grad(o, leaves, do)
    assert th.equal(o, v) and th.equal(dv, do)
    for got, other in ((dq, k), (dk_, q)):
        size = (do.float() * v.float()).abs().view(-1, dk).sum(-1).max() * other.float().abs().max()
        assert got.float().abs().max() <= 2 * dk * U * size
    more = th.zeros(n + 1, 1, heads * dk, device="cuda", dtype=th.bfloat16)
    with pytest.raises(ValueError, match="unsupported shape"):
        pkg.cross_attention(more, more, more, heads)
