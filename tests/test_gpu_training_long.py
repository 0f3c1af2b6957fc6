"""Training on clips that one block's LDS does not hold: the model's attention changes to the tiles of
cross_attention there (...training.attention), at the operator and through a whole step."""
import math

import pytest
import torch as th

from oracle import ref_denoiser
from tests.conftest import oracle_cfg

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tr(pkg):
    import importlib
    return importlib.import_module(pkg.__name__ + ".training")


# on both sides of the border: the whole backward pass in LDS (first), the forward pass alone, neither; above 256 rows
@pytest.mark.parametrize("lq,lk,dk", [(111, 111, 64), (112, 112, 64), (150, 40, 64), (40, 257, 32), (257, 40, 32), (300, 301, 32)])
def test_attention_on_both_sides_of_the_lds(tr, lq, lk, dk):
    n, heads = 2, 3
    g = th.Generator().manual_seed(lq + lk)
    q, k, v, do = (th.randn(n, rows, heads * dk, generator=g) for rows in (lq, lk, lk, lq))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = tr.attention(*leaves, heads, 1 / math.sqrt(dk))
    o.backward(do.cuda())
    with th.no_grad():
        again = tr.attention(*leaves, heads, 1 / math.sqrt(dk))
    ts = [t.double().reshape(n, -1, heads, dk).transpose(1, 2).requires_grad_(True) for t in (q, k, v)]
    p = th.softmax(ts[0] @ ts[1].transpose(-1, -2) / math.sqrt(dk), -1)
    want = (p @ ts[2]).transpose(1, 2).reshape(n, lq, heads * dk)
    want.backward(do.double())
    # f32: a score is a sum of dk products of size up to ~4 sqrt(dk), off by at most (dk + 2) 2^-24 of
    # their absolute sum, |q|.|k| scale <= ~ sqrt(dk) * 2: 64 terms * 2^-24 * 16 = 6e-5 at worst, on top the
    # sums over up to 301 rows of values up to ~4 and 8: 301 * 2^-24 = 2e-5.  Relative to the largest value: 2e-4.
    for got, exact in [(o, want), (again, want)] + [(a.grad, b.grad.transpose(1, 2).reshape(n, -1, heads * dk)) for a, b in zip(leaves, ts)]:
        exact = exact.detach()
        assert (got.detach().cpu().double() - exact).abs().max() <= 2e-4 * exact.abs().max()


def test_a_step_on_long_clips_matches_the_oracle(tr, pkg, beat_cfg):
    """160 frames over the memory of 128000 samples: the loss and every gradient against autograd through the
    oracle's model.  The bounds are those of the 40-frame step (1e-5 of the loss, 2e-3 of a tensor's largest
    gradient, or of 1e-4 of the model's largest): each is relative, a step's chain of operators is as long, and only
    the sums over frames have 4 times the terms, whose rounding grows by less than that from 2^-24."""
    poses, L, n = 123, 160, 2
    arch = pkg.arch_from_config(beat_cfg.Model, poses)
    sd = pkg.init_state_dict(arch, seed=0, perturb=True)
    encoder, _, _, _, _ = pkg.create_model(poses, beat_cfg.Model, dtype="f32", device="cuda:0")
    encoder.load_state_dict(sd)
    diffusion = pkg.create_diffusion(beat_cfg.Model.Diffusion.to_dict(), True)
    g = th.Generator().manual_seed(11)
    z = encoder.encoder()((th.randn(n, 128000, generator=g) * 0.1).cuda())
    model = tr.TrainableModel(arch, sd, "cuda")
    x0, noise, t = th.randn(n, poses, L, generator=g), th.randn(n, poses, L, generator=g), th.tensor([873, 12])
    model.zero_grad()
    loss = tr.training_losses(diffusion, model, x0.cuda(), t.cuda(), {"speech_tokens": z}, noise=noise.cuda())["mse"].mean()
    loss.backward()

    names = list(model.params)
    sd_ref = {k: v.detach().float().clone().requires_grad_(k in model.params) for k, v in sd.items()}
    ca, cb = (th.from_numpy(a[t.numpy()]).float().reshape(-1, 1, 1)
              for a in (diffusion.sqrt_alphas_cumprod, diffusion.sqrt_one_minus_alphas_cumprod))
    cfg = oracle_cfg(arch)
    speech = ref_denoiser.speech_memory(sd_ref, cfg, tuple(a.cpu() for a in z))
    eps = ref_denoiser.denoise(sd_ref, cfg, ca * x0 + cb * noise, t, speech=speech)
    want = ((eps - noise) ** 2).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    floor = 1e-4 * max(sd_ref[k].grad.abs().max().item() for k in names)
    for k in names:
        a, b = model.params[k].grad.cpu(), sd_ref[k].grad
        assert (a - b).abs().max().item() <= 2e-3 * max(b.abs().max().item(), floor), k
