"""CPU tests of the decoder-block operators (…_amd/blocks.py): the buckets' plan, the C structure's layout, and every
refusal, in Python and at the C entries, none of which launches anything."""
import copy
import ctypes
import importlib
import math
import os
import pickle
import subprocess

import numpy as np
import pytest
import torch as th

from tests.conftest import ROOT


@pytest.fixture(scope="module")
def native(pkg):
    return importlib.import_module(pkg.__name__ + ".native")


@pytest.mark.parametrize("n_buckets,most,both", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (20, 200, True), (64, 2047, True),
                                                 (8, 5, True), (1024, 2000, True)])
def test_relative_buckets(pkg, n_buckets, most, both):
    """The definition over the reals: a distance at a border opens its bucket (its logarithm in 64 bits may not say so)."""
    b = pkg.RelativeBuckets(n_buckets, most, both, device="cpu").buckets
    side = n_buckets // 2 if both else n_buckets
    near = side // 2
    steps = side - near
    assert b.dtype == th.int32 and b.numel() == 2 * most + 1
    for d in range(-most, most + 1):
        far = abs(d) if both else max(0, -d)
        if far < near:
            want = far
        else:
            x = math.log(far / near) / math.log(most / near) * steps
            k = round(x) if abs(x - round(x)) < 1e-9 else math.floor(x)
            if abs(x - round(x)) < 1e-9:   # a border in 64 bits: whole numbers decide
                k = round(x) if far ** steps >= near ** (steps - round(x)) * most ** round(x) else round(x) - 1
            want = near + min(k, steps - 1)
        assert b[d + most] == want + (side if both and d > 0 else 0), d
    assert b.min() == 0 and b.max() <= n_buckets - 1


def test_relative_buckets_refusals(pkg):
    for args in ((0, 8), (3, 8, True), (2, 8, True), (1, 8, False), (32, 8, True), (8, 2048, True), (1026, 2000, True), (32, 16, False)):
        with pytest.raises(ValueError):
            pkg.RelativeBuckets(*args, device="cpu")


def test_operators_refuse_host_tensors(pkg):
    """No CPU fallback."""
    x = th.zeros(1, 2, 8)
    with pytest.raises(ValueError):
        pkg.cross_attention(x, x, x, 2)
    with pytest.raises(ValueError):
        pkg.relative_attention(x, x, x, 2, pkg.RelativeBuckets(8, 16, device="cpu"), th.zeros(8, 2))
    with pytest.raises(ValueError):
        pkg.residual_norm(x, x, (th.ones(8), None))
    with pytest.raises(ValueError):
        pkg.cross_attention(None, x, x, 2)


def test_struct_layout_matches_header(native, tmp_path):
    fields = [f for f, _ in native.BattnArgs._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ggd_train.h"\nint main(void) {\n' +
                   "".join(f'printf("%zu\\n", offsetof(ggd_tr_battn_args, {f}));\n' for f in fields) +
                   'printf("%zu\\n", sizeof(ggd_tr_battn_args));\nreturn 0;\n}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(native.BattnArgs, f).offset for f in fields] + [ctypes.sizeof(native.BattnArgs)]


def _battn(native, **over):
    """Arguments in order for 2 clips, with addresses that a refused call never touches."""
    at = 1 << 20
    d = dict(n=2, heads=4, kv_heads=2, lq=3, lk=5, dk=16, dtype=1, scale=0.25, q=at, k=at, v=at, o=at, ldq=64, bq=192, ldk=32, bk=160, ldv=32,
             bv=160, ldo=64, bo=192, stat=at, o32=at, dout=at, dq=at, dk_out=at, dv=at, ws=at, ws_bytes=1 << 40)
    d.update(over)
    return native.BattnArgs(**d)


BAD = [dict(n=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(lq=0), dict(lk=0), dict(dk=0), dict(dtype=2), dict(dtype=-1), dict(scale=0.0),
       dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(ldq=-1), dict(bk=-8), dict(q=None), dict(k=None), dict(v=None),
       dict(table=1 << 20), dict(buckets=1 << 20), dict(table=1 << 20, buckets=1 << 20, n_buckets=0, distance=4),
       dict(table=1 << 20, buckets=1 << 20, n_buckets=4, distance=0)]
UNSUPPORTED = [dict(dk=129), dict(lq=(1 << 28) + 1), dict(lk=(1 << 28) + 1), dict(table=1 << 20, buckets=1 << 20, n_buckets=1025, distance=4),
               dict(table=1 << 20, buckets=1 << 20, n_buckets=8, distance=2048), dict(n=1 << 20, lq=1 << 20), dict(n=1, heads=64, kv_heads=1, lq=1 << 27),
               dict(n=1 << 30, heads=1 << 30, kv_heads=1 << 30, lq=1 << 28),   # (a product past 64 bits)
               dict(n=1, heads=1 << 17, kv_heads=1 << 17, table=1 << 20, buckets=1 << 20, n_buckets=1024, distance=2047)]


def test_attention_entry_refusals(native):
    lib = native.load()
    call = lambda fn, **over: fn(ctypes.byref(_battn(native, **over)), None)
    for over in BAD:
        assert call(lib.ggd_tr_battn_fwd, **over) == -1, over
        assert call(lib.ggd_tr_battn_bwd, **over) == -1, over
    for over in UNSUPPORTED:
        assert call(lib.ggd_tr_battn_fwd, **over) == -2, over
        assert call(lib.ggd_tr_battn_bwd, **over) == -2, over
        assert lib.ggd_tr_battn_ws(ctypes.byref(_battn(native, **over)), 1) == 0
    assert lib.ggd_tr_battn_fwd(None, None) == -1 and lib.ggd_tr_battn_bwd(None, None) == -1 and lib.ggd_tr_battn_ws(None, 0) == 0
    for over in (dict(o=None), dict(stat=None), dict(o32=None), dict(stat=(1 << 20) + 4)):
        assert call(lib.ggd_tr_battn_fwd, **over) == -1, over
    long = dict(lq=1, lk=100000)   # divided among blocks: needs its workspace
    need = lib.ggd_tr_battn_ws(ctypes.byref(_battn(native, **long)), 0)
    assert need > 0
    for over in (dict(ws=None), dict(ws=(1 << 20) + 8), dict(ws_bytes=need - 1)):
        assert call(lib.ggd_tr_battn_fwd, **long, **over) == -1, over
    need = lib.ggd_tr_battn_ws(ctypes.byref(_battn(native)), 1)
    for over in (dict(stat=None), dict(o32=None), dict(dout=None), dict(dq=None), dict(dk_out=None), dict(dv=None), dict(ws=None),
                 dict(ws_bytes=need - 1), dict(dtable=1 << 20), dict(stat=(1 << 20) + 4)):
        assert call(lib.ggd_tr_battn_bwd, **over) == -1, over
    assert call(lib.ggd_tr_battn_fwd, n=0) == 0 and call(lib.ggd_tr_battn_bwd, n=0) == 0


def test_residual_norm_entry_refusals(native):
    lib = native.load()
    at = 1 << 20
    names = ("rows", "d", "dtype", "kind", "scale", "eps", "h", "y", "gate", "gate_rows", "post_g", "post_b", "pre_g", "pre_b")
    good = dict(rows=6, d=8, dtype=0, kind=0, scale=1.0, eps=1e-5, h=at, y=at, gate=at, gate_rows=3, post_g=at, post_b=at, pre_g=at, pre_b=at)

    def fwd(h_out=at, u=at, **over):
        d = dict(good, **over)
        return lib.ggd_tr_resnorm_fwd(*(d[k] for k in names), h_out, u, at, None)

    outs = dict(stats=at, dh_out=at, du=at, dh=at, dy=at, dgate=at, d_post_g=at, d_post_b=at, d_pre_g=at, d_pre_b=at, ws=at, ws_bytes=1 << 40)

    def bwd(**over):
        d = dict(good, **{k: v for k, v in over.items() if k in good})
        o = dict(outs, **{k: v for k, v in over.items() if k in outs})
        return lib.ggd_tr_resnorm_bwd(*(d[k] for k in names), *o.values(), None)

    for over in (dict(rows=-1), dict(d=0), dict(dtype=2), dict(kind=2), dict(eps=0.0), dict(eps=math.nan), dict(gate_rows=0), dict(gate_rows=4),
                 dict(pre_g=None), dict(post_g=None), dict(h=None), dict(y=None)):
        assert fwd(**over) == -1, over
        assert bwd(**over) == -1, over
    for over in (dict(h_out=None), dict(u=None)):
        assert fwd(**over) == -1, over
    for over in (dict(d=8193), dict(rows=1 << 32, gate=None)):
        assert fwd(**over) == -2, over
        assert bwd(**dict(over, dgate=None if "gate" in over else at)) == -2, over
    for over in (dict(rows=0), *({k: None} for k in outs if k != "ws_bytes"), dict(gate=None), dict(pre_b=None), dict(post_b=None), dict(ws=at + 8),
                 dict(ws_bytes=lib.ggd_tr_resnorm_ws(6, 8, 3, 1) - 1)):
        assert bwd(**over) == -1, over
    assert fwd(rows=0) == 0
    assert lib.ggd_tr_resnorm_ws(0, 8, 1, 0) == 0 and lib.ggd_tr_resnorm_ws(6, 8, 4, 1) == 0 and lib.ggd_tr_resnorm_ws(6, 8193, 3, 1) == 0


def test_entries_are_declared(native):
    for name in ("ggd_tr_resnorm_fwd", "ggd_tr_resnorm_bwd", "ggd_tr_resnorm_ws", "ggd_tr_battn_fwd", "ggd_tr_battn_bwd", "ggd_tr_battn_ws"):
        assert name in native.EXPORTS


def test_forward_mode_derivatives_are_refused(pkg):
    """A tangent would be lost: NotImplementedError, whichever operand carries it, with reverse-mode gradients or without."""
    fw = th.autograd.forward_ad
    x, w, table = th.ones(1, 2, 8), th.ones(8), th.zeros(8, 2)
    buckets = pkg.RelativeBuckets(8, 16, device="cpu")
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, th.ones_like(t))
        for call in (lambda: pkg.cross_attention(dual(x), x, x, 2), lambda: pkg.cross_attention(x, dual(x), x, 2), lambda: pkg.cross_attention(x, x, dual(x), 2),
                     lambda: pkg.cross_attention(dual(x.clone().requires_grad_()), x, x, 2),
                     lambda: pkg.relative_attention(x, x, x, 2, buckets, dual(table)),
                     lambda: pkg.residual_norm(dual(x), x, (w, None)), lambda: pkg.residual_norm(x, dual(x), (w, None)),
                     lambda: pkg.residual_norm(x, x, (dual(w), None)), lambda: pkg.residual_norm(x, x, (w, dual(w))),
                     lambda: pkg.residual_norm(x, x, (w, None), post=(dual(w), None)), lambda: pkg.residual_norm(x, x, (w, None), post=(w, dual(w))),
                     lambda: pkg.residual_norm(x, x, (w, None), gate=dual(w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with th.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_tracing_is_refused(pkg):
    """A trace would hold the outputs' allocations without the kernels: NotImplementedError under every tracer, and for
    tensors without memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w = th.ones(1, 2, 8), th.ones(8)
    table, buckets = th.zeros(8, 2), pkg.RelativeBuckets(8, 16, device="cpu")
    for call in (lambda t: pkg.cross_attention(t, t, t, 2), lambda t: pkg.relative_attention(t, t, t, 2, buckets, table),
                 lambda t: pkg.residual_norm(t, t, (w, None))[1]):
        with pytest.raises(NotImplementedError, match="traced"):
            th.jit.trace(call, (x,))
        for mode in ("real", "fake", "symbolic"):
            with pytest.raises(NotImplementedError, match="traced"):
                make_fx(call, tracing_mode=mode)(x)
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(call, pre_dispatch=True)(x)
        with FakeTensorMode() as mode:
            fake = th.empty(1, 2, 8, device="cuda")
            with pytest.raises(NotImplementedError, match="traced"):
                call(fake)
        with pytest.raises(NotImplementedError, match="traced"):
            call(fake)


@pytest.mark.parametrize("dtype,heads,dk", [(1, 3 << 16, 128), (0, 3 << 15, 128), (0, 3 << 16, 64), (1, 3 << 19, 9), (0, 3 << 19, 5)])
def test_rows_too_wide_for_their_offsets_are_unsupported(native, dtype, heads, dk):
    """A tile has 64 rows, whose byte offsets are 32-bit numbers: 63 rows' width past 2^31 would wrap, and rows of another place or zeros be
    read.  (The workspace is left out, so that an entry that takes the shape answers -1 and launches nothing.)"""
    lib = native.load()
    size = 4 if dtype == 0 else 2
    width = heads * ((dk * size + 15) // 16 * 16)
    assert 63 * width + 16 * ((dk * size + 15) // 16) > (1 << 31) - 1
    most = _battn(native, n=0, heads=(1 << 31) - 1, kv_heads=1, dk=dk, dtype=dtype)   # (no clip: refused by the width alone)
    assert lib.ggd_tr_battn_fwd(ctypes.byref(most), None) == -2
    for over, want in ((dict(heads=heads), -2), (dict(heads=heads // 2), -1)):
        args = _battn(native, n=1, kv_heads=1, lq=64, lk=64, dk=dk, dtype=dtype, ldq=8, bq=8, ldk=8, bk=8, ldv=8, bv=8, ws=None, ws_bytes=0, **over)
        assert lib.ggd_tr_battn_bwd(ctypes.byref(args), None) == want
        args.ldq = 1 << 23   # packed
        assert lib.ggd_tr_battn_fwd(ctypes.byref(args), None) == want
        assert (lib.ggd_tr_battn_ws(ctypes.byref(args), 1) > 0) == (want == -1)


def test_long_memories_are_limited_by_the_launches_they_need(native):
    """8 clips of 32 heads over 3 million states (17 hours at 50 a second): the forward pass has no block a key, the backward pass one of
    128 keys a kv head.  (The workspace is left out: an entry that takes the shape answers -1 and launches nothing.)"""
    lib = native.load()
    shape = dict(n=8, heads=32, kv_heads=8, lq=1, dk=16, ldq=512, bq=512, ldk=128, ldv=128, bk=1 << 40, bv=1 << 40, ldo=512, bo=512, ws=None, ws_bytes=0)
    for lk, stat, want in ((3000000, None, -1), (3000000, 1 << 20, -1), (1 << 28, None, -1), (1 << 23, 1 << 20, -1), ((1 << 23) + 1, 1 << 20, -2)):
        args = _battn(native, lk=lk, stat=stat, o32=stat, **shape)
        assert lib.ggd_tr_battn_fwd(ctypes.byref(args), None) == want, (lk, stat)
        assert (lib.ggd_tr_battn_ws(ctypes.byref(args), 0) > 0) == (want == -1)
        args = _battn(native, lk=lk, **shape)
        assert lib.ggd_tr_battn_bwd(ctypes.byref(args), None) == (-1 if lk <= 1 << 23 else -2)


def test_an_operand_out_of_line_is_packed_alone(native):
    """The workspace holds the rows that are laid out anew: of the one operand that is not in whole aligned 16-byte units."""
    lib = native.load()
    need = lambda backward, **over: lib.ggd_tr_battn_ws(ctypes.byref(_battn(native, **dict(dict(lk=300, bk=9600, bv=9600), **over))), backward)
    at, q, k = 1 << 20, 2 * 3 * 4 * 16 * 2, 2 * 300 * 2 * 16 * 2   # bytes of q's rows and of k's
    up = lambda x: (x + 255) // 256 * 256
    for backward in (0, 1):
        plain = need(backward)
        for over, more in ((dict(q=at + 2), up(q)), (dict(ldq=68, bq=204), up(q)), (dict(k=at + 8), up(k)), (dict(v=at + 4, bv=9601), up(k)),
                           (dict(q=at + 2, k=at + 2), up(q) + up(k)), (dict(dout=at + 6), up(q) if backward else 0)):
            assert need(backward, **over) - plain == more, over
        odd = dict(dk=15, ldq=60, ldk=30, ldv=30)
        assert need(backward, **odd) >= (2 if backward else 1) * up(q) + 2 * up(k)


def test_partial_sums_of_many_gate_rows_stay_few(native):
    """Blocks of the backward pass, and with them the partial sums, are bounded whatever the number of gate rows, each of 2 to 7 rows; a count
    past any limit of a launch is no other case."""
    lib = native.load()
    for d in (64, 1024, 1032, 8192):
        for groups in (1, 1000, 1025, 4097, 100000, (1 << 22) + 1, (1 << 28)):
            for rows in (2, 7):
                blocks = lib.ggd_tr_resnorm_ws(groups * rows, d, rows, 1) / (5 * d * 4)
                assert 0 < blocks <= 4096, (d, groups, rows, blocks)
        assert lib.ggd_tr_resnorm_ws(1 << 30, d, 1, 0) / (5 * d * 4) <= 1024


def test_gate_sum_entry_refusals(native):
    lib = native.load()
    at = 1 << 20

    def call(sizes, kept, src=at, dtype=1, out=at, ws=None, ws_bytes=0, axes=None):
        n = len(sizes)
        return lib.ggd_tr_gate_sum(n if axes is None else axes, (ctypes.c_int64 * n)(*sizes), (ctypes.c_uint8 * n)(*kept), src, dtype, out, ws, ws_bytes, None)

    def need(sizes, kept):
        n = len(sizes)
        return lib.ggd_tr_gate_sum_ws(n, (ctypes.c_int64 * n)(*sizes), (ctypes.c_uint8 * n)(*kept))

    for bad in (dict(src=None), dict(out=None), dict(dtype=2), dict(axes=-1)):
        assert call((2, 3), (1, 0), **bad) == -1, bad
    assert call((2, 0), (1, 0)) == -1 and call((2, -3), (1, 0)) == -1 and call((1 << 40, 1 << 40), (1, 0)) == -1
    assert lib.ggd_tr_gate_sum(2, None, None, at, 1, at, None, 0, None) == -1
    assert call((2,) * 18, (1, 0) * 9) == -2 and need((2,) * 18, (1, 0) * 9) == 0
    # axes of one kind in a row, and those of size 1, count as one: long sums of few outputs are divided
    long = ((1, 3, 50, 1, 400, 2), (1, 0, 0, 1, 0, 1))
    parts = need(*long) // (2 * 4)
    assert parts > 1 and call(*long) == -1 and call(*long, ws=at, ws_bytes=need(*long) - 1) == -1
    assert need((1 << 31, 64), (1, 0)) == 0 and need((1 << 20, 5), (0, 1)) == 1024 * 5 * 4


def test_backward_without_the_memorys_gradients(native):
    """dk and dv both null: a valid call, without the workspace of their parts.  (ws left out: nothing is launched.)"""
    lib = native.load()
    shape = dict(n=1, heads=2, kv_heads=2, lq=2000, lk=300, dk=64, ldq=128, bq=256000, ldk=128, bk=38400, ldv=128, bv=38400, ldo=128, bo=256000)
    need = [lib.ggd_tr_battn_ws(ctypes.byref(_battn(native, **shape, **over)), 1) for over in ({}, dict(dk_out=None, dv=None))]
    assert 0 < need[1] < need[0]
    for over in (dict(dk_out=None), dict(dv=None), dict(dk_out=None, dv=None, dq=None), dict(dk_out=None, dv=None, ws_bytes=need[1] - 1)):
        assert lib.ggd_tr_battn_bwd(ctypes.byref(_battn(native, **shape, **over)), None) == -1, over


def test_arguments_of_another_kind_are_refused(pkg):
    """ValueError, as documented, whatever an argument is; and no number is cut to a whole one."""
    x, w = th.zeros(1, 2, 8), th.ones(8)
    plan, table = pkg.RelativeBuckets(8, 16, device="cpu"), th.zeros(8, 2)
    assert pkg.RelativeBuckets(np.int64(8), np.int32(16), device="cpu").buckets.equal(plan.buckets)
    for call in (lambda: pkg.RelativeBuckets(8.0, 16, device="cpu"), lambda: pkg.RelativeBuckets(8, 16.9, device="cpu"),
                 lambda: pkg.RelativeBuckets("8", 16, device="cpu"), lambda: pkg.RelativeBuckets(None, device="cpu")):
        with pytest.raises(ValueError, match="whole number"):
            call()
    for over in (dict(heads="2"), dict(heads=2.5), dict(heads=None), dict(kv_heads=1.5), dict(scale="1"), dict(scale=x), dict(mask=[[True, True]]),
                 dict(mask=1), dict(q_mask="all")):
        args = dict(dict(heads=2), **over)
        with pytest.raises(ValueError, match="has to be a tensor|whole numbers"):
            pkg.cross_attention(x, x, x, **args)
    for offset in (1.5, "1", None, x):
        with pytest.raises(ValueError, match="offset"):
            pkg.relative_attention(x, x, x, 2, plan, table, offset=offset)
    for over, match in ((dict(pre=(1.0, None)), "tensors"), (dict(pre=("w", None)), "tensors"), (dict(gate=0.5), "tensors"), (dict(post=(w, 0)), "tensors"),
                        (dict(kind=["layer"]), "layer or rms"), (dict(kind=None), "layer or rms"), (dict(scale="x"), "scale"), (dict(scale=None), "scale"),
                        (dict(eps=w), "eps"), (dict(pre=w[0]), "weight, bias")):
        with pytest.raises(ValueError, match=match):
            pkg.residual_norm(x, x, **dict(dict(pre=(w, None)), **over))


def test_the_binding_belongs_to_one_torch(native, monkeypatch):
    """Another torch than the binding was built against: it counts as stale, and is not bound."""
    if native.is_stale():
        native.build()
    assert not native._binding_is_stale() and native.load_blocks().torch_version == th.__version__
    monkeypatch.setattr(th, "__version__", "0.1")
    assert native._binding_is_stale() and native.is_stale()
    monkeypatch.setattr(native, "_blocks", None)
    with pytest.raises(ImportError, match="torch"):
        native.load_blocks()
    monkeypatch.undo()
    monkeypatch.setattr(native, "BINDING_TORCH", native.BINDING_TORCH + ".none")
    assert native._binding_is_stale()


def test_a_plan_is_copied_without_its_devices(pkg):
    """A loaded or copied plan makes its own copies on devices: those of another process, moved elsewhere on loading, would be read where
    they are not."""
    plan = pkg.RelativeBuckets(8, 16, device="cpu")
    plan._on[th.device("cuda", 0)] = plan.on("cpu")   # what torch.load(..., map_location="cpu") made of a copy on a GPU
    for other in (pickle.loads(pickle.dumps(plan)), copy.deepcopy(plan)):
        assert other._on == {} and other.buckets.equal(plan.buckets) and (other.n_buckets, other.max_distance, other.both_sides) == (8, 16, True)
