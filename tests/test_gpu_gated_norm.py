"""GPU tests of the norms around a token branch (gated_norm_fwd / gated_norm_bwd) against the formulas in 64 bits.

Tolerances, relative to the largest value of the output, from what is rounded.  A bfloat16 output is rounded once:
2^-8 relative to the value itself, and n or a gradient inherits fp32 errors that are far below.  float32: a row sum of C
terms in fp32 (tree of lanes, at most 16 + log2 terms deep each) is off by less than (16 + 10) 2^-24 of the sum of
magnitudes; it enters n and the gradients through mean, rstd and the two projections, each at most a factor 8 on these
inputs (rows of deviation 1 around a mean below 8): 8 * 26 * 2^-24 * 4 < 5e-5.  Column sums of M terms are kept in fp32
by each lane over at most M / 64 rows and in double across workgroups: below 1e-4 of the sum of magnitudes for the M
used here.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def make(shape, seed, dt, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale + mean).to(dt)


def formula(x, f, gate, keep, scale, post, pre, kind, eps, dr=None, dn=None):
    """64-bit outputs and, with dr / dn, the gradients by autograd of the definition."""
    lv = {}

    def leaf(k, t):
        if t is None:
            return None
        lv[k] = t.detach().double().cpu().requires_grad_(True)
        return lv[k]

    def normed(v, w, b):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w
        return v if b is None else v + b
    X, Fv = leaf("x", x), leaf("f", f)
    g = leaf("gate", gate)
    po = None if post is None else (leaf("post_weight", post[0]), leaf("post_bias", post[1]))
    pr = None if pre is None else (leaf("pre_weight", pre[0]), leaf("pre_bias", pre[1]))
    h = Fv if po is None else normed(Fv, *po)
    if g is not None:
        h = h * g
    if keep is not None:
        B = keep.numel()
        h = (h.reshape(B, -1) * keep.double().cpu()[:, None]).reshape(h.shape)
    r = scale * X + h
    n = None if pr is None else normed(r, *pr)
    grads = None
    if dr is not None or dn is not None:
        loss = 0.0
        if dr is not None:
            loss = loss + (r * dr.double().cpu()).sum()
        if dn is not None:
            loss = loss + (n * dn.double().cpu()).sum()
        grads = dict(zip(lv, torch.autograd.grad(loss, list(lv.values()), allow_unused=True)))
    return r.detach(), None if n is None else n.detach(), grads


def close(got, want, dt, what, extra=1.0):
    got, want = got.detach().double().cpu(), want.double()
    assert torch.isfinite(got).all(), what
    big = want.abs().max().clamp_min(1e-30)
    tol = 5e-5 * extra * big + (2.0 ** -8 * want.abs() if dt == BF else 0.0)
    bad = ((got - want).abs() - tol).max().item()
    assert bad <= 0, (what, bad, big.item())


def check(shape, dt, kind="layer", post=True, gate=True, pre=True, samples=0, scale=1.0, bias=True, dr=True, seed=0,
          x=None, f=None):
    from unet_amd import ops
    C = shape[-1]
    x = make(shape, seed + 1, dt, 1.0, 0.5) if x is None else x
    f = make(shape, seed + 2, dt, 0.7, -0.2) if f is None else f
    po = (make(C, seed + 3, F32, 0.2, 1.0), make(C, seed + 4, F32, 0.2) if bias else None) if post else None
    pr = (make(C, seed + 5, F32, 0.2, 1.0), make(C, seed + 6, F32, 0.2) if bias else None) if pre else None
    g = make(C, seed + 7, F32, 0.3, 0.5) if gate else None
    keep = (make(samples, seed + 8, F32).sign() + 1.0) * 0.6 if samples else None
    d1 = make(shape, seed + 9, dt, 0.1) if dr else None
    d2 = make(shape, seed + 10, dt, 0.1) if pre else None
    cu = lambda t: None if t is None else t.cuda()
    pair = lambda p: None if p is None else (cu(p[0]), cu(p[1]))
    kw = dict(gate=cu(g), keep=cu(keep), res_scale=scale, post=pair(po), pre=pair(pr), kind=kind, eps=1e-5)
    X, Fv = (t if t.is_cuda else t.cuda() for t in (x, f))
    r, n, stats = ops.gated_norm_fwd(X, Fv, **kw)
    wr, wn, wg = formula(x, f, g, keep, scale, po, pr, kind, 1e-5, d1, d2)
    close(r, wr, dt, "r")
    assert (n is None) == (pr is None)
    if n is not None:
        close(n, wn, dt, "n")
    r2, _, none = ops.gated_norm_fwd(X, Fv, want_stats=False, **kw)
    assert none is None and torch.equal(r, r2)
    got = ops.gated_norm_bwd(cu(d1), cu(d2), X, Fv, stats, **kw)
    again = ops.gated_norm_bwd(cu(d1), cu(d2), X, Fv, stats, **kw)
    for name in got._fields:
        t, want = getattr(got, name), wg.get(name)
        assert (t is None) == (name not in wg), name
        if t is not None:
            want = torch.zeros_like(t, dtype=torch.float64).cpu() if want is None else want
            close(t, want, dt if name in ("x", "f") else F32, name, extra=4.0)
            assert torch.equal(t, getattr(again, name)), name


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [1, 2, 7, 8, 31, 32, 33, 64, 96, 100, 128, 192, 255, 384, 512, 513, 768, 1001, 1024, 2040,
                               2048, 2049, 4096, 4104, 5003, 8191, 8192])
def test_widths(C, dt):
    check((3, 5, C), dt, samples=3)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 64, 65, 1000, 4099])
def test_row_counts(rows, dt):
    check((rows, 96), dt)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("pre", [False, True])
def test_parts(kind, post, gate, pre):
    for dt in (F32, BF):
        check((4, 9, 160), dt, kind, post, gate, pre, samples=4, scale=0.75)
        check((36, 77), dt, kind, post, gate, pre, bias=False)


def test_without_the_residual_streams_gradient():
    check((4, 9, 160), BF, dr=False)
    check((4, 9, 161), F32, "rms", dr=False, post=False)


@pytest.mark.parametrize("C", [96, 384, 1024, 4096])
def test_more_rows_than_workgroups(C):
    check(((1 << 20) // C * 8 + 3, C), BF)


def test_strided_and_unaligned_rows():
    for dt in (F32, BF):
        wide = make((2, 7, 3 * 96), 1, dt).cuda()
        check((2, 7, 96), dt, x=wide[..., 96:192], f=wide[..., 192:])
        odd = make((14, 3 * 96 + 1), 2, dt).cuda()      # rows off 16 bytes
        check((14, 96), dt, x=odd[:, 1:97], f=odd[:, 97:193])
        flat = make(14 * 96 + 3, 3, dt).cuda()          # a base off 16 bytes
        check((14, 96), dt, x=flat[3:].view(14, 96))


def test_rows_far_from_zero_and_constant_rows():
    from unet_amd import ops
    C = 192
    w, b = torch.ones(C).cuda(), torch.zeros(C).cuda()
    x = make((64, C), 1, F32).cuda()
    far = x + 4096.0
    _, n, _ = ops.gated_norm_fwd(far, torch.zeros_like(x), pre=(w, b))
    want = torch.nn.functional.layer_norm(far.double(), (C,))
    # x + 4096 is rounded on input (the same for both); the row mean is off by less than 26 * 2^-24 * 4096
    assert (n.double() - want).abs().max() < 26 * 2.0 ** -24 * 4096 * 2
    flat = torch.full((5, C), 3.0).cuda()
    r, n, st = ops.gated_norm_fwd(flat, torch.zeros_like(flat), pre=(w, b))
    assert torch.equal(r, flat) and n.abs().max().item() == 0.0      # 3 * 192 / 192 is exact
    d = ops.gated_norm_bwd(None, torch.ones_like(flat), flat, torch.zeros_like(flat), st, pre=(w, b))
    assert torch.isfinite(d.x).all()


def test_dropped_samples_pass_the_stream_through():
    from unet_amd import ops
    x, f = make((4, 6, 96), 1, BF).cuda(), make((4, 6, 96), 2, BF).cuda()
    keep = torch.tensor([0.0, 1.25, 0.0, 1.0]).cuda()
    g = make(96, 3, F32).cuda()
    po = (torch.ones(96).cuda(), None)
    r, _, st = ops.gated_norm_fwd(x, f, gate=g, keep=keep, post=po)
    assert torch.equal(r[0], x[0]) and torch.equal(r[2], x[2])
    d = ops.gated_norm_bwd(x, None, x, f, st, gate=g, keep=keep, post=po)
    assert d.f[0].abs().max() == 0 and d.f[2].abs().max() == 0 and d.f[1].abs().max() > 0


def test_gradients_against_differences():
    from unet_amd import ops
    C, M = 40, 6
    x, f = make((M, C), 1, F32).cuda(), make((M, C), 2, F32).cuda()
    ps = {"gate": make(C, 3, F32, 0.3, 1.0).cuda(), "qw": make(C, 4, F32, 0.3, 1.0).cuda(), "qb": make(C, 5, F32).cuda(),
          "pw": make(C, 6, F32, 0.3, 1.0).cuda(), "pb": make(C, 7, F32).cuda(), "x": x, "f": f}
    dr, dn = make((M, C), 8, F32).cuda(), make((M, C), 9, F32).cuda()

    def run(p):
        return ops.gated_norm_fwd(p["x"], p["f"], gate=p["gate"], post=(p["qw"], p["qb"]), pre=(p["pw"], p["pb"]), res_scale=0.5)

    def loss(p):
        r, n, _ = run(p)
        return ((r.double() * dr).sum() + (n.double() * dn).sum()).item()
    st = run(ps)[2]
    d = ops.gated_norm_bwd(dr, dn, x, f, st, gate=ps["gate"], post=(ps["qw"], ps["qb"]), pre=(ps["pw"], ps["pb"]), res_scale=0.5)
    got = {"gate": d.gate, "qw": d.post_weight, "qb": d.post_bias, "pw": d.pre_weight, "pb": d.pre_bias, "x": d.x, "f": d.f}
    for k, t in ps.items():
        v = make(tuple(t.shape), 20, F32).cuda()
        e = 2.0 ** -7
        num = (loss({**ps, k: t + e * v}) - loss({**ps, k: t - e * v})) / (2 * e)
        ana = (got[k].double() * v).sum().item()
        # third-order term of the central difference (e^2 times O(1) third derivatives over 240 elements) and the
        # fp32 rounding of two losses of magnitude ~100 over 2 e
        assert abs(num - ana) < 240 * e * e + 100 * 2.0 ** -20 / e, (k, num, ana)


def test_no_rows():
    from unet_amd import ops
    x = torch.empty((0, 96), dtype=BF, device="cuda")
    w = torch.ones(96).cuda()
    r, n, st = ops.gated_norm_fwd(x, x, gate=w, pre=(w, w))
    assert r.shape == n.shape == (0, 96)
    d = ops.gated_norm_bwd(x, x, x, x, st, gate=w, pre=(w, w))
    assert d.x.shape == (0, 96) and d.gate.abs().max() == 0 and d.pre_bias.abs().max() == 0


def test_rows_past_two_gigabytes():
    """Row offsets beyond 32 bits: a wide row stride puts the last rows past 2^32 bytes."""
    from unet_amd import ops
    C, ld, M = 96, 1 << 20, 2200
    big = torch.empty((M, ld), dtype=BF, device="cuda")
    x = big[:, 64:64 + C]
    x.copy_(make((M, C), 1, BF).cuda())
    f = make((M, C), 2, BF).cuda()
    w = torch.ones(C).cuda()
    r, n, st = ops.gated_norm_fwd(x, f, pre=(w, None))
    r2, n2, st2 = ops.gated_norm_fwd(x.contiguous(), f, pre=(w, None))
    assert torch.equal(r, r2) and torch.equal(n, n2) and torch.equal(st, st2)


def test_other_stream_and_graph_replay():
    from unet_amd import ops
    M, C = 777, 384
    x, f, dr, dn = (make((M, C), i, BF).cuda() for i in range(4))
    g, w, b = make(C, 5, F32).cuda(), make(C, 6, F32).cuda(), make(C, 7, F32).cuda()
    kw = dict(gate=g, post=(w, b), pre=(w, b))

    def step():
        r, n, st = ops.gated_norm_fwd(x, f, **kw)
        return (r, n) + tuple(ops.gated_norm_bwd(dr, dn, x, f, st, **kw))
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.cuda.graph(other):
        out2 = step()
    for k in range(4):
        x.copy_(make((M, C), 30 + k, BF).cuda())
        want = step()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
        assert all(torch.equal(a, b) for a, b in zip(out2, want)), k


def test_refusals():
    from unet_amd import ops
    x = torch.zeros((4, 96), dtype=BF, device="cuda")
    w = torch.ones(96).cuda()
    st = torch.zeros((4, 4)).cuda()
    bad = [lambda: ops.gated_norm_fwd(x, x[:, :48]), lambda: ops.gated_norm_fwd(x, x.float()),
           lambda: ops.gated_norm_fwd(x.half(), x.half()), lambda: ops.gated_norm_fwd(x.t(), x.t()),
           lambda: ops.gated_norm_fwd(x, x, gate=w[:95]), lambda: ops.gated_norm_fwd(x, x, gate=w.bfloat16()),
           lambda: ops.gated_norm_fwd(x, x, gate=w.cpu()), lambda: ops.gated_norm_fwd(x, x, pre=(None, w)),
           lambda: ops.gated_norm_fwd(x, x, keep=torch.ones(3).cuda()), lambda: ops.gated_norm_fwd(x, x, kind="batch"),
           lambda: ops.gated_norm_fwd(torch.zeros((1, 8193)).cuda(), torch.zeros((1, 8193)).cuda()),
           lambda: ops.gated_norm_fwd(x[:1].expand(4, 96), x),
           lambda: ops.gated_norm_bwd(x, x, x, x, st), lambda: ops.gated_norm_bwd(None, None, x, x, st),
           lambda: ops.gated_norm_bwd(x, None, x, x, st, pre=(w, None)), lambda: ops.gated_norm_bwd(x, None, x, x, st[:3]),
           lambda: ops.gated_norm_bwd(x[:, :48], None, x, x, st), lambda: ops.gated_norm_bwd(x.float(), None, x, x, st)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError):
        ops.gated_norm_fwd(x.cpu(), x.cpu())
