"""GPU tests of the gated norms, the 4-bit products and the SwinUNet options built on them, at the edges: norms with
different eps, infinities and NaN, inputs that want a gradient, 4-bit weights whose parameters have changed.

Tolerances are those of the operators' and the model's own tests: gated norms float32 5e-5 of the largest value (20e-5 for
gradients: four times as many sums), bfloat16 2^-8 of the value more; float32 models 1e-4 relative L2, gradients 2e-2.
Infinities and NaN have to stand where the definition in 64 bits has them.
"""
import pytest
import torch
import torch.nn.functional as F

from oracle import swin_oracle
from oracle import weights as W

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def make(shape, seed, dt=F32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale + mean).to(dt)


def rel(a, b):
    a, b = a.detach().double().cpu().reshape(-1), b.detach().double().cpu().reshape(-1)
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def formula(x, f, dr, dn, gate=None, post=None, pre=None, kind="layer", post_eps=1e-5, pre_eps=1e-5):
    """(r, n, gradients by name) in 64 bits; the gradients by autograd of the definition."""
    lv = {}

    def leaf(k, t):
        if t is None:
            return None
        lv[k] = t.detach().double().cpu().requires_grad_(True)
        return lv[k]

    def normed(v, w, b, eps):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w
        return v if b is None else v + b
    h = leaf("f", f)
    X, g = leaf("x", x), leaf("gate", gate)
    if post is not None:
        h = normed(h, leaf("post_weight", post[0]), leaf("post_bias", post[1]), post_eps)
    r = X + (h if g is None else h * g)
    n = None if pre is None else normed(r, leaf("pre_weight", pre[0]), leaf("pre_bias", pre[1]), pre_eps)
    outs = [t for t in (r, n) if t is not None]
    grads = torch.autograd.grad(outs, list(lv.values()), [t.double().cpu() for t in (dr, dn) if t is not None])
    return r.detach(), None if n is None else n.detach(), dict(zip(lv, grads))


def agree(got, want, dt, what, extra=1.0):
    """Equal infinities and NaN; finite values within the tolerance."""
    got, want = got.detach().double().cpu(), want.detach().double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(torch.nan_to_num(got[~fin]), torch.nan_to_num(want[~fin])), what
    big = want[fin].abs().max().clamp_min(1e-30)
    tol = 5e-5 * extra * big + (2.0 ** -8 * want[fin].abs() if dt == BF else 0.0)
    bad = ((got[fin] - want[fin]).abs() - tol).max().item()
    assert bad <= 0, (what, bad, big.item())


def check_norm(x, f, dr, dn, dt, names=None, rows=None, **kw):
    """Both directions of the gated norm against the formula.  names: the gradients to look at (all of them), rows: which
    rows of dx and df."""
    from unet_amd import ops
    cu = lambda t: None if t is None else t.cuda()
    pair = lambda p: None if p is None else (cu(p[0]), cu(p[1]))
    eps = (kw.get("post_eps", 1e-5), kw.get("pre_eps", 1e-5))
    a = dict(gate=cu(kw.get("gate")), post=pair(kw.get("post")), pre=pair(kw.get("pre")), kind=kw.get("kind", "layer"),
             eps=eps if eps[0] != eps[1] else eps[0])
    r, n, st = ops.gated_norm_fwd(x.cuda(), f.cuda(), **a)
    wr, wn, wg = formula(x, f, dr, dn, **kw)
    agree(r, wr, dt, "r")
    if wn is not None:
        agree(n, wn, dt, "n")
    got = ops.gated_norm_bwd(cu(dr), cu(dn), x.cuda(), f.cuda(), st, **a)
    for name in got._fields:
        t = getattr(got, name)
        assert (t is None) == (name not in wg), name
        if t is not None and (names is None or name in names):
            of_rows = name in ("x", "f")
            t, want = (v[rows] if of_rows and rows is not None else v for v in (t.cpu(), wg[name]))
            agree(t, want, dt if of_rows else F32, name, 4.0)


# ------------------------------------------------------------------ the two norms' eps
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [77, 96, 1024])
def test_each_norm_has_its_own_eps(C, dt, kind):
    x, f = make((37, C), 1, dt, 0.3), make((37, C), 2, dt, 0.2)
    for bias in (True, False):
        vec = lambda s, m: make(C, s, F32, 0.2, m)
        post, pre = (vec(3, 1.0), vec(4, 0.0) if bias else None), (vec(5, 1.0), vec(6, 0.0) if bias else None)
        for pe, ne in ((0.25, 1e-5), (1e-5, 0.5), (0.1, 0.01), (0.03, 0.03)):
            check_norm(x, f, make((37, C), 8, dt, 0.1), make((37, C), 9, dt, 0.1), dt, gate=vec(7, 0.5), post=post, pre=pre,
                       kind=kind, post_eps=pe, pre_eps=ne)


def norm_eps(name):
    """An eps for a norm of a block: four different ones a block, others in the next."""
    at = sum(int(c) for c in name if c.isdigit())
    return (0.02, 0.3, 0.05, 0.11, 0.2)[(at + 2 * ("post" in name)) % 5]


def gated_block(sd, pre, x, H, Wd, heads, ws, shift, mask, keep1=None, keep2=None):
    """A block with norms behind its branches and gates, each norm with norm_eps of its name."""
    B, L, C = x.shape
    ln = lambda v, k: F.layer_norm(v, (C,), sd[pre + k + ".weight"], sd[pre + k + ".bias"], norm_eps(pre + k))

    def branch(f, which, keep):
        f = ln(f, f"post_norm{which}") * sd[pre + f"gate{which}"]
        return f if keep is None else f * keep.view(B, 1, 1).to(f.dtype)
    h = ln(x, "norm1").view(B, H, Wd, C)
    He, We = max(H, ws), max(Wd, ws)
    h = F.pad(h, (0, 0, 0, We - Wd, 0, He - H))
    if shift > 0:
        h = torch.roll(h, (-shift, -shift), (1, 2))
    a = swin_oracle.window_attention(sd, pre + "attn.", swin_oracle._partition(h, ws), heads, ws,
                                     None if mask is None else mask.to(x.dtype))
    h = swin_oracle._unpartition(a, ws, He, We)
    if shift > 0:
        h = torch.roll(h, (shift, shift), (1, 2))
    x = x + branch(h[:, :H, :Wd, :].reshape(B, L, C), 1, keep1)
    y = F.linear(ln(x, "norm2"), sd[pre + "mlp.0.weight"], sd[pre + "mlp.0.bias"])
    y = F.linear(F.gelu(y), sd[pre + "mlp.3.weight"], sd[pre + "mlp.3.bias"])
    return x + branch(y, 2, keep2)


def swin(dt, **options):
    from unet_amd.swin import SwinUNet
    cfg = dict(swin_oracle.DEFAULT_CONFIG, **options)
    m = SwinUNet(cfg, compute_dtype=dt)
    sd = W.fill_state_dict(swin_oracle.swin_template(cfg), seed=42)
    for i, (k, v) in enumerate(m.state_dict().items()):
        if k not in sd:
            base = cfg["layer_scale"] if "gate" in k else 1.0 if k.endswith("weight") else 0.0
            sd[k] = make(tuple(v.shape), 100 + i, F32, 0.2 * (base or 1.0), base)
    m.load_state_dict(sd)
    return m.cuda(), sd, cfg


def test_a_gated_model_honours_every_norms_eps(monkeypatch):
    monkeypatch.setattr(swin_oracle, "swin_block", gated_block)
    m, sd, cfg = swin(F32, post_norm=True, layer_scale=0.5)
    used = set()
    for name, mod in m.named_modules():
        if ".blocks." in name and isinstance(mod, torch.nn.LayerNorm):
            mod.eps = norm_eps(name)
            used.add((name.split(".")[1], name.split(".")[3], mod.eps))
    assert sum(t[:2] == ("0", "0") for t in used) == 4      # four different ones in a block
    x, y, _ = W.synthetic_batch(3, 4, 64, 64, seed=42)
    assert rel(m.eval()(x.cuda()), swin_oracle.swin_unet_forward(sd, x, cfg, False)[0]) < 1e-4
    m.train()
    drop = [[None, None]] * sum(cfg["depths"])
    m.drop_path_override = drop
    out = m(x.cuda())
    tgt = F.adaptive_avg_pool2d(y, out.shape[-2:])
    ((out - tgt.cuda()) ** 2).mean().backward()
    leaves = {k: v.double().requires_grad_(True) for k, v in sd.items() if v.is_floating_point() and "running_" not in k}
    full = {k: leaves.get(k, v.double() if v.is_floating_point() else v) for k, v in sd.items()}
    ref, _ = swin_oracle.swin_unet_forward(full, x.double(), cfg, True, drop)
    ((ref - tgt.double()) ** 2).mean().backward()
    assert rel(out, ref) < 1e-3      # (training mode: batch statistics over few elements)
    got = dict(m.named_parameters())
    num = sum(((got[k].grad.double().cpu() - t.grad) ** 2).sum() for k, t in leaves.items())
    den = sum((t.grad ** 2).sum() for t in leaves.values())
    assert (num / den).sqrt().item() < 2e-2
    for k, t in leaves.items():
        if ("gate" in k or "post_norm" in k or ".norm" in k) and t.grad.norm() > 1e-7 * den.sqrt():
            assert rel(got[k].grad, t.grad) < 5e-2, k


# ------------------------------------------------------------------ infinities and NaN
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("C", [77, 96, 4096])
def test_an_infinite_column_sum_stays_infinite_without_a_bias(C, kind):
    """dgate = w sum(u fhat) + b sum(u): without b there is no second term, and infinity times nothing is not NaN."""
    x, f, dr = make((40, C), 1), make((40, C), 2), make((40, C), 3)
    dr[7, 5], dr[20, C - 1] = float("inf"), float("-inf")
    w, gate = make(C, 4, F32, 0.2, 1.0), make(C, 5, F32, 0.2, 0.5)
    want = formula(x, f, dr, None, gate=gate, post=(w, None), kind=kind)[2]
    assert torch.isinf(want["gate"]).sum() == 2 and torch.isinf(want["post_weight"]).sum() == 2
    # (behind a norm the two rows' own gradients are infinities added and subtracted: what of them is NaN is no one's)
    rows = [i for i in range(40) if i not in (7, 20)]
    check_norm(x, f, dr, None, F32, rows=rows, gate=gate, post=(w, None), kind=kind)
    check_norm(x, f, dr, None, F32, gate=gate, kind=kind)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [77, 96, 8192])
def test_an_infinite_gate_without_a_bias_behind_it(C, dt):
    x, f, dr = make((5, C), 1, dt), make((5, C), 2, dt), make((5, C), 3, dt)
    w, gate = make(C, 4, F32, 0.2, 1.0), make(C, 5, F32, 0.2, 0.5)
    gate[3], gate[C - 1] = float("inf"), float("-inf")
    assert torch.isinf(formula(x, f, dr, None, gate=gate)[0]).sum() == 10
    check_norm(x, f, dr, None, dt, gate=gate)
    # (infinities of both signs are added up in what flows back through a norm)
    check_norm(x, f, dr, None, dt, names=("x", "gate"), gate=gate, post=(w, None))
    check_norm(x, f, dr, make((5, C), 6, dt), dt, names=(), gate=gate, pre=(w, None), kind="rms")


@pytest.mark.parametrize("M", [1, 3, 17, 63])
@pytest.mark.parametrize("C", [24, 96, 200])
def test_an_infinite_last_row_counts_once(M, C):
    """Workgroups of several rows, the last of them short: the rows that are not there add nothing, whatever the last holds."""
    x, f, dr = make((M, C), 1), make((M, C), 2), make((M, C), 3).abs()
    f[M - 1, 2], f[M - 1, C - 1] = float("inf"), float("-inf")
    gate = make(C, 5, F32, 0.2, 0.5)
    assert torch.isinf(formula(x, f, dr, None, gate=gate)[2]["gate"]).sum() == 2
    check_norm(x, f, dr, None, F32, gate=gate)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("C", [77, 96, 512])
def test_nan_and_infinite_rows_stay_alone(C, dt):
    from unet_amd import ops
    x, f, dr, dn = (make((70, C), i, dt) for i in range(4))
    f[69, 0], x[3, C - 1], f[40, 5], dr[50, 1] = float("nan"), float("inf"), float("-inf"), float("nan")
    w, b, gate = make(C, 4, F32, 0.2, 1.0).cuda(), make(C, 6).cuda(), make(C, 5, F32, 0.2, 0.5).cuda()
    kw = dict(gate=gate, post=(w, b), pre=(w, b))
    r, n, st = ops.gated_norm_fwd(x.cuda(), f.cuda(), **kw)
    assert (~torch.isfinite(n)).any(1).nonzero().flatten().tolist() == [3, 40, 69]
    assert (~torch.isfinite(r)).any(1).nonzero().flatten().tolist() == [3, 40, 69]
    d = ops.gated_norm_bwd(dr.cuda(), dn.cuda(), x.cuda(), f.cuda(), st, **kw)
    for t in (d.x, d.f):
        assert (~torch.isfinite(t)).any(1).nonzero().flatten().tolist() == [3, 40, 50, 69]
    keep = [i for i in range(70) if i not in (3, 40, 50, 69)]
    y = ops.gated_norm_bwd(dr[keep].cuda(), dn[keep].cuda(), x[keep].cuda(), f[keep].cuda(), st[keep].contiguous(), **kw)
    assert torch.equal(d.x[keep], y.x) and torch.equal(d.f[keep], y.f)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("rows,K,N", [(20, 300, 40), (600, 1000, 700), (1100, 200, 130), (3400, 900, 3100)])
def test_gelu_of_infinities(rows, K, N, dt):
    """v Phi(v) at -infinity is infinity times nothing: NaN, in either type and every kernel; +infinity stays, and a large
    negative number is nothing."""
    from unet_amd import ops
    x, qw, bias = make((rows, K), 1, dt).cuda(), ops.mx_quantize(make((N, K), 2, F32, K ** -0.5).cuda()), make(N, 3).cuda()
    plain = ops.mx_linear(x, qw, bias=bias, act=2)
    bias[1], bias[N - 1], bias[5] = float("-inf"), float("inf"), -3e38
    y = ops.mx_linear(x, qw, bias=bias, act=2)
    assert torch.isnan(y[:, 1]).all() and (y[:, N - 1] == float("inf")).all() and (y[:, 5].abs() < 1e-6).all()
    rest = [i for i in range(N) if i not in (1, 5, N - 1)]
    assert torch.equal(y[:, rest], plain[:, rest])


# ------------------------------------------------------------------ inputs that want a gradient
def test_4_bit_operators_refuse_what_wants_a_gradient():
    from unet_amd import ops
    for dt in (F32, BF):
        x, w, b = make((6, 96), 1, dt).cuda(), make((40, 96), 2).cuda(), make(40, 3).cuda()
        res, out = make((6, 40), 4, dt).cuda(), torch.empty((6, 40), dtype=dt, device="cuda")
        qw, qx = ops.mx_quantize(w), ops.mx_quantize(x)
        want = ops.mx_linear(x, qw, bias=b, resid=res)
        leaf = lambda t: t.detach().clone().requires_grad_(True)
        calls = [lambda: ops.mx_linear(leaf(x), qw, bias=b, resid=res), lambda: ops.mx_linear(x, qw, bias=leaf(b), resid=res),
                 lambda: ops.mx_linear(x, qw, bias=b, resid=leaf(res)), lambda: ops.mx_linear(qx, qw, bias=b, resid=leaf(res), dtype=dt),
                 lambda: ops.mx_linear(qx, qw, bias=leaf(b), resid=res, dtype=dt),
                 lambda: ops.mx_linear(x, qw, bias=b, resid=res, out=leaf(out)),
                 lambda: ops.mx_linear(x, ops.mx_quantize(leaf(w)), bias=b, resid=res),
                 lambda: ops.mx_linear(ops.mx_quantize(leaf(x)), qw, bias=b, resid=res, dtype=dt)]
        for i, f in enumerate(calls):
            with pytest.raises(RuntimeError, match="gradient"):
                f()
                pytest.fail(f"call {i} was not refused")
            with torch.no_grad():
                assert torch.equal(f(), want), i


# ------------------------------------------------------------------ 4-bit weights whose parameters have changed
def quantised_model(dt=BF, **options):
    m, sd, cfg = swin(dt, **options)
    x = W.synthetic_batch(1, 4, 64, 64, seed=42)[0].cuda()
    m.eval().quantize_linears()
    return m, x


def replace_by_loading(m):
    m.load_state_dict({k: v * 1.5 if v.is_floating_point() else v for k, v in m.state_dict().items()}, assign=True)


def replace_parameter(m):
    w = m.layers[0].blocks[1].mlp[0].weight
    m.layers[0].blocks[1].mlp[0].weight = torch.nn.Parameter(w.detach() * 1.5)


def replace_module(m):
    old = m.layers[1].blocks[0].attn.proj
    m.layers[1].blocks[0].attn.proj = torch.nn.Linear(old.in_features, old.out_features).to(old.weight.device)


def replace_block(m):
    from unet_amd.swin import SwinTransformerBlock
    b = m.layers[1].blocks[0]
    m.layers[1].blocks[0] = SwinTransformerBlock(b.dim, b.num_heads, b.window_size, b.shift_size, b.mlp_ratio).cuda().eval()


@pytest.mark.parametrize("change", [replace_by_loading, replace_parameter, replace_module, replace_block])
def test_replaced_parameters_are_refused_until_quantised_again(change):
    m, x = quantised_model()
    with torch.no_grad():
        a = m(x)
        change(m)
        with pytest.raises(RuntimeError, match="quantize_linears"):
            m(x)
        assert not torch.equal(m.quantize_linears()(x), a)
        assert torch.equal(m(x), m(x))


def test_optimizer_steps_replayed_from_the_callers_own_graph_are_seen():
    import unet_amd
    m, x = quantised_model()
    opt = unet_amd.FusedAdamW(m.parameters(), lr=1e-2, capturable=True)
    for i, p in enumerate(m.parameters()):
        p.grad = make(tuple(p.shape), i, F32, 0.1).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            opt.step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    with torch.no_grad():
        b = m.quantize_linears()(x)
        assert torch.equal(m(x), b)
        for _ in range(3):
            graph.replay()
            with pytest.raises(RuntimeError, match="quantize_linears"):
                m(x)
            c = m.quantize_linears()(x)
            assert not torch.equal(b, c)
            b = c
        # a loaded optimizer state puts its step count back: still seen
        sd = opt.state_dict()
        graph.replay()
        opt.load_state_dict(sd)
        with pytest.raises(RuntimeError, match="quantize_linears"):
            m(x)


def test_a_captured_4_bit_prediction_follows_the_next_quantisation():
    """The 4-bit weights stay where a captured forward pass reads them."""
    m, x = quantised_model()
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                m(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="relaxed"):
            out = m(x)
        for k in range(4):
            want = m(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), k
            for layer in m.layers:
                for blk in layer.blocks:
                    blk.mlp[3].weight.mul_(1.25)
            if k == 2:      # (back and again: still the same memory)
                m.dequantize_linears()
                torch.cuda.synchronize()
            m.quantize_linears()


def test_a_captured_step_takes_an_optimizer_that_wraps_the_fused_one():
    import unet_amd
    from unet_amd.graph import GraphedTrainStep
    x, y, _ = W.synthetic_batch(1, 4, 64, 64, seed=42)
    m, _, cfg = swin(F32)
    m.train()
    m.drop_path_override = [[None, None]] * sum(cfg["depths"])
    inner = unet_amd.FusedAdamW(m.parameters(), lr=1e-3, capturable=True)

    class Wrapper:
        capturable = True
        zero_grad, step, sync_hyper = inner.zero_grad, inner.step, inner.sync_hyper
        snapshot, restore = inner.snapshot, inner.restore
    loss = lambda out, label: ((out - F.interpolate(label, out.shape[-2:])) ** 2).mean()
    step = GraphedTrainStep(m, loss, Wrapper(), x.cuda(), y.cuda(), warmup=2)
    with torch.no_grad():
        a = m.eval().quantize_linears()(x.cuda())
        for _ in range(2):
            step(x.cuda(), y.cuda())
            with pytest.raises(RuntimeError, match="quantize_linears"):
                m(x.cuda())
        assert not torch.equal(m.quantize_linears()(x.cuda()), a)
    assert inner.device_step_count() == 2


def test_weights_are_quantised_again_in_and_out_of_inference_mode():
    m, x = quantised_model()
    with torch.inference_mode():
        want = m(x).clone()
        m.quantize_linears()
    with torch.no_grad():
        assert torch.equal(m(x), want)
    m.dequantize_linears()
    fresh, _ = quantised_model()
    fresh.dequantize_linears()
    fresh._mx_kept = None
    with torch.inference_mode():
        fresh.quantize_linears()      # (memory that was made in inference mode)
    fresh.quantize_linears()
    with torch.no_grad():
        assert torch.equal(fresh(x), want)


def test_quantisation_into_memory_that_is_there():
    from unet_amd import ops
    for dt in (F32, BF):
        a, b = make((70, 200), 1, dt).cuda(), make((70, 200), 2, dt).cuda()
        q, want = ops.mx_quantize(a), ops.mx_quantize(b)
        at = q.data.data_ptr()
        assert ops.mx_quantize(b, out=q) is q and q.data.data_ptr() == at and torch.equal(q.data, want.data)
        for bad in (a[:, :199], a[:64], a.view(7, 10, 200)):
            with pytest.raises(ValueError, match="out"):
                ops.mx_quantize(bad, out=q)
        with pytest.raises(TypeError, match="out"):
            ops.mx_quantize(a, out=b)


def test_a_gradient_sink_gets_the_gradients_of_every_parameter():
    m, _, cfg = swin(BF, post_norm=True, layer_scale=0.5)
    x = W.synthetic_batch(2, 4, 64, 64, seed=42)[0].cuda()
    m.train()
    m.drop_path_override = [[None, None]] * sum(cfg["depths"])
    m(x).square().mean().backward()
    plain = {k: p.grad.clone() for k, p in m.named_parameters()}
    m.zero_grad(set_to_none=True)
    seen = {}

    def sink(name, t):
        seen[name] = t.clone()      # (on the stream that made it)
        return t
    m.grad_sink = sink
    m(x).square().mean().backward()
    torch.cuda.synchronize()
    for k in plain:
        assert torch.equal(seen[k], plain[k]), k


def test_4_bit_prediction_in_float32():
    """With a float32 compute type the pass quantises the same way; the two types' outputs differ by the bfloat16 pass's
    roundings and by the 4 bits that these turn over, and by far less than a wrong product would make of it."""
    m, x = quantised_model(F32)
    with torch.no_grad():
        q = m(x)
        assert q.dtype == F32 and torch.isfinite(q).all() and torch.equal(m(x), q)
        assert not torch.equal(m.dequantize_linears()(x), q)


def test_a_copied_model_is_refused_until_quantised_by_itself():
    import copy
    m, x = quantised_model()
    with torch.no_grad():
        a = m(x)
        other = copy.deepcopy(m)
        with pytest.raises(RuntimeError, match="quantize_linears"):
            other(x)
        other.layers[0].blocks[0].mlp[0].weight.mul_(1.5)
        assert not torch.equal(other.quantize_linears()(x), a)
        assert torch.equal(m(x), a)      # (nothing is shared between the two)
        assert torch.equal(m.quantize_linears()(x), a)


def test_blocks_added_between_two_quantisations_are_quantised():
    from unet_amd.swin import SwinTransformerBlock
    m, x = quantised_model()
    n = len(m._mx_linears)
    with torch.no_grad():
        m(x)
        b = m.layers[1].blocks[0]
        m.layers[1].blocks.append(SwinTransformerBlock(b.dim, b.num_heads, b.window_size, 0, b.mlp_ratio).cuda().eval())
        m.quantize_linears()
        assert len(m._mx_linears) == n + 4
        want = m(x)
        m._mx_kept = None      # (into fresh memory)
        assert torch.equal(m.quantize_linears()(x), want)
