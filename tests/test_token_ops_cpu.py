"""CPU tests of the gated norms' and 4-bit products' entry points: sizes, and refusals before anything is launched (the
pointers below are never read)."""
import pytest
import torch

from unet_amd import _lib, ops

P = 1 << 20      # an aligned address that nothing reads


def lib():
    return _lib.load()


def refused(name, *args, match):
    with pytest.raises(ValueError, match=match):
        _lib.call(name, *args)


def test_sizes():
    assert lib().unetk_gated_norm_max_channels() == ops._NORM_MAX_C
    # units of 64 rows x 128 k: 4096 bytes of codes, 256 of scales
    for rows, K, units in ((1, 1, 1), (64, 128, 1), (65, 128, 2), (64, 129, 2), (1000, 1000, 16 * 8)):
        assert lib().unetk_mx_codes_bytes(rows, K) == units * 4096
        assert lib().unetk_mx_scales_bytes(rows, K) == units * 256
    for rows, K in ((0, 5), (5, 0), (-1, 5), (1 << 31, 5), (5, 1 << 21)):
        assert lib().unetk_mx_codes_bytes(rows, K) == 0
    # partial rows of the backward pass: no more than the rows there are, and no more than the chip holds
    assert lib().unetk_gated_norm_bwd_rows(1, 96) == 1
    assert lib().unetk_gated_norm_bwd_rows(1 << 20, 96) == 768
    assert lib().unetk_gated_norm_bwd_rows(1 << 20, 8192) == 256
    assert lib().unetk_gated_norm_bwd_rows(0, 96) == 0 and lib().unetk_gated_norm_bwd_rows(5, 8193) == 0
    # activations are quantised inside the product for a few rows and for short K under many rows
    ws = lib().unetk_mx_linear_x_workspace_bytes
    assert ws(1, 4096, 4096, _lib.BF16) == 0 and ws(4096, 96, 384, _lib.F32) == 0
    assert ws(1, 4095, 4096, _lib.BF16) > 0      # a row that is no whole 16-byte pieces
    assert ws(300, 1000, 64, _lib.BF16) == (5 * 8) * (4096 + 256)


def norm_fwd(x=P, ldx=96, f=P, ldf=96, gate=None, keep=None, rps=0, qw=None, qb=None, pw=None, pb=None, r=P, n=None, M=4, C=96,
             dt=1):
    return (x, ldx, f, ldf, gate, keep, rps, 1.0, qw, qb, pw, pb, 0, 1e-5, r, n, None, M, C, dt, None)


@pytest.mark.parametrize("kw,match", [(dict(dt=2), "dtype"), (dict(C=0, ldx=0, ldf=0), "C=0"), (dict(C=8193, ldx=9000, ldf=9000), "C=8193"),
                                      (dict(M=0), "rows"), (dict(M=1 << 31), "rows"), (dict(x=None), "null"), (dict(r=None), "null"),
                                      (dict(ldx=95), "overlapping"), (dict(keep=P, rps=3), "samples"), (dict(keep=P, rps=0), "samples"),
                                      (dict(pw=P), "norm in front"), (dict(n=P), "norm in front"), (dict(qb=P), "without its weight"),
                                      (dict(pb=P), "without its weight")])
def test_norm_forward_refuses(kw, match):
    refused("unetk_gated_norm_fwd", *norm_fwd(**kw), match=match)


def norm_bwd(dr=P, dn=None, stats=P, gate=None, qw=None, qb=None, pw=None, dg=None, dqw=None, dqb=None, dpw=None, dpb=None, lddr=96,
             partials=P, M=4, C=96):
    return (dr, lddr, dn, 96, P, 96, P, 96, stats, gate, None, 0, 1.0, qw, qb, pw, 0, P, P, dg, dqw, dqb, dpw, dpb, partials, M, C, 1,
            None)


@pytest.mark.parametrize("kw,match", [(dict(stats=None), "null"), (dict(partials=None), "null"), (dict(dr=None), "null"),
                                      (dict(lddr=90), "overlapping"), (dict(pw=P), "norm in front"), (dict(dn=P), "norm in front"),
                                      (dict(dg=P), "not there"), (dict(dqw=P), "not there"), (dict(qb=P), "not there"),
                                      (dict(dpb=P), "not there"), (dict(M=0), "rows"), (dict(C=9000, lddr=9000), "C=9000")])
def test_norm_backward_refuses(kw, match):
    refused("unetk_gated_norm_bwd", *norm_bwd(**kw), match=match)


@pytest.mark.parametrize("args,match", [((None, 96, 4, 96, 1, P, P), "null"), ((P, 96, 4, 96, 1, P + 4, P), "misaligned"),
                                        ((P, 96, 4, 96, 1, P, P + 8), "misaligned"), ((P, 95, 4, 96, 1, P, P), "overlapping"),
                                        ((P, 96, 0, 96, 1, P, P), "matrix"), ((P, 96, 4, 96, 5, P, P), "dtype"),
                                        ((P, 1 << 20, 1 << 30, 1 << 20, 1, P, P), "matrix")])
def test_quantise_refuses(args, match):
    refused("unetk_mx_quantize", *args, None, match=match)


def linear(xc=P, xs=P, wc=P, ws=P, out=P, ldo=40, M=4, K=96, N=40, act=0, resid=None, ldr=0, dt=1):
    return (xc, xs, wc, ws, out, ldo, M, K, N, None, act, resid, ldr, dt, None)


@pytest.mark.parametrize("kw,match", [(dict(xc=None), "null"), (dict(wc=None), "null"), (dict(xs=P + 4), "misaligned"),
                                      (dict(ws=P + 4), "misaligned"), (dict(ldo=39), "overlapping"), (dict(resid=P, ldr=39), "overlapping"),
                                      (dict(act=1), "activation"), (dict(act=3), "activation"), (dict(dt=7), "dtype"),
                                      (dict(M=0), "matrix"), (dict(K=0), "matrix"), (dict(N=1 << 25, ldo=1 << 25), "outputs")])
def test_product_refuses(kw, match):
    refused("unetk_mx_linear", *linear(**kw), match=match)


def test_product_of_unquantised_rows_refuses():
    refused("unetk_mx_linear_x", None, 96, P, P, P, 40, 4, 96, 40, None, 0, None, 0, 1, None, None, match="null")
    refused("unetk_mx_linear_x", P, 95, P, P, P, 40, 4, 96, 40, None, 0, None, 0, 1, None, None, match="overlapping")
    refused("unetk_mx_linear_x", P, 1000, P, P, P, 40, 300, 1000, 40, None, 0, None, 0, 1, None, None, match="workspace")


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 96), torch.zeros(96)
    for f in (lambda: ops.gated_norm_fwd(x, x, pre=(w, w)), lambda: ops.mx_quantize(x)):
        with pytest.raises(RuntimeError, match="GPU"):
            f()


def test_steps_of_an_optimizer_are_known_to_its_parameters():
    import unet_amd
    from unet_amd.optim import steps_taken
    a, b = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    one = unet_amd.FusedAdamW([a], lr=1e-3)
    two = unet_amd.FusedAdamW([{"params": [a]}], lr=1e-3)
    two.add_param_group({"params": [b]})
    assert steps_taken(a) == steps_taken(b) == steps_taken(torch.zeros(1)) == 0
    one.step()      # (no gradient is there: nothing is launched)
    assert (steps_taken(a), steps_taken(b)) == (1, 0)
    two.step()
    two.step()
    assert (steps_taken(a), steps_taken(b)) == (3, 2)


@pytest.mark.parametrize("rows", [1, 2, 5])
def test_shared_memory_is_seen(rows):
    """Against the set of bytes that each operand covers."""
    for lda in (4, 6, 9):
        for ldb in (4, 6, 9):
            for ca in (1, 3, 4):
                for cb in (1, 2, 4):
                    for b in range(0, 60):
                        a = 20
                        one = {a + r * lda + c for r in range(rows) for c in range(ca)}
                        two = {b + r * ldb + c for r in range(rows) for c in range(cb)}
                        apart = ops._apart(a, ca, b, cb, rows, lda, ldb)
                        if lda == ldb or rows == 1:
                            # (one gap behind the last row may count as shared)
                            assert apart <= (not one & two) and (apart or one & two or abs(b - a) <= rows * lda), (lda, ldb, ca, cb, b)
                        else:
                            assert apart <= (not one & two)
