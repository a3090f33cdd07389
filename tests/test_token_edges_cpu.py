"""CPU tests of what surrounds the gated norms and the 4-bit weights: which eps reaches which norm, refusals before
anything is launched, and what counts as a change of a parameter."""
import pytest
import torch

from unet_amd import _lib, ops

P = 1 << 20      # an aligned address that nothing reads


def test_a_gated_block_passes_each_norms_eps():
    from unet_amd.swin import SwinTransformerBlock, _gated_args
    blk = SwinTransformerBlock(96, 3, 8, post_norm=True, layer_scale=0.1)
    blk.norm1.eps, blk.post_norm1.eps, blk.norm2.eps, blk.post_norm2.eps = 1.0, 2.0, 3.0, 4.0
    nxt = torch.nn.LayerNorm(96, eps=5.0)
    assert _gated_args(blk, 1, blk.norm2)["eps"] == (2.0, 3.0)
    assert _gated_args(blk, 2, nxt)["eps"] == (4.0, 5.0)
    assert _gated_args(blk, 2, None)["eps"][0] == 4.0
    gates = SwinTransformerBlock(96, 3, 8, layer_scale=0.1)
    gates.norm2.eps = 3.0
    assert _gated_args(gates, 1, gates.norm2)["eps"][1] == 3.0


def norm_fwd(x=P, ldx=96, f=P, ldf=96, keep=None, rps=0, qw=None, qb=None, pw=None, pb=None, r=P, n=None, M=4, C=96, dt=1):
    return (x, ldx, f, ldf, None, keep, rps, 1.0, qw, qb, pw, pb, 0, 1e-5, 1e-6, r, n, None, M, C, dt, None)


@pytest.mark.parametrize("kw,match", [(dict(dt=2), "dtype"), (dict(C=8193, ldx=9000, ldf=9000), "C=8193"), (dict(M=0), "rows"),
                                      (dict(x=None), "null"), (dict(ldf=95), "overlapping"), (dict(keep=P, rps=3), "samples"),
                                      (dict(pw=P), "norm in front"), (dict(n=P), "norm in front"), (dict(qb=P), "without its weight")])
def test_norm_forward_with_two_eps_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _lib.call("unetk_gated_norm_fwd_eps", *norm_fwd(**kw))


def test_steps_that_a_device_counter_took_are_counted():
    """A step captured by the caller is replayed without Python: its count is the device's (a host tensor stands for it here).
    It only ever grows, also where a loaded state puts the device's back."""
    import unet_amd
    from unet_amd.optim import steps_taken
    a = torch.nn.Parameter(torch.zeros(3))
    opt = unet_amd.FusedAdamW([a], lr=1e-3, capturable=True)
    opt.step()      # (no gradient is there: nothing is launched)
    hyper = torch.tensor([5.0, 1e-3, 0.0, 0.9, 0.999], dtype=torch.float64)
    opt._hyper[0] = [hyper, None, (1e-3, 1e-2, 0.9, 0.999)]
    opt._steps.append(hyper)
    before = steps_taken(a)
    hyper[0] += 2
    assert steps_taken(a) == before + 2
    seen = {before + 2}
    for _ in range(3):      # steps, then back to an earlier state
        hyper[0] += 1
        assert steps_taken(a) not in seen
        seen.add(steps_taken(a))
        opt.load_state_dict({"state": {}, "param_groups": opt.state_dict()["param_groups"]})
        assert hyper[0] == 0 and steps_taken(a) not in seen
        seen.add(steps_taken(a))


def test_broadcast_parameters_count_as_changed(monkeypatch):
    """The broadcast writes past autograd's version counter; what is derived from a parameter and kept beside it (4-bit
    weights) goes by that counter."""
    from unet_amd import dist as udist
    m = torch.nn.Linear(3, 2)
    monkeypatch.setattr(udist.dist, "is_initialized", lambda: True)
    monkeypatch.setattr(udist.dist, "get_world_size", lambda *a: 2)
    monkeypatch.setattr(udist.dist, "broadcast", lambda t, src: t.data.fill_(7.0))
    before = [p._version for p in m.parameters()]
    udist.broadcast_parameters(m)
    assert all((p == 7.0).all() for p in m.parameters())
    assert all(p._version != v for p, v in zip(m.parameters(), before))
