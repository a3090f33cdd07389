"""GPU tests of SwinUNet with norms behind the branches, gates on them, and 4-bit linears in prediction: the whole model
against the CPU oracle with its block extended by the two options.

Tolerances are those of the plain model's tests: float32 outputs 1e-4 relative L2, gradients 2e-2 against float64 (batch
statistics over few elements in the decoder); bfloat16 eval 2e-2.
"""
import pytest
import torch
import torch.nn.functional as F

from oracle import swin_oracle
from oracle import weights as W

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.detach().double().cpu().reshape(-1), b.detach().double().cpu().reshape(-1)
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def mx(t):
    """Values of t's rows in microscaled 4 bits, in t's type."""
    K = t.shape[-1]
    b = F.pad(t.detach().double().reshape(-1, K), (0, -K % 32)).view(-1, (K + 31) // 32, 32)
    big = b.abs().amax(-1, keepdim=True)
    scale = torch.pow(2.0, torch.where(big > 0, torch.frexp(big)[1] - 3, -127).double())
    y = b / scale
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    q = (torch.round(y / step) * step).clamp(-6, 6) * scale
    return q.view(-1, b.shape[1] * 32)[:, :K].reshape(t.shape).to(t.dtype)


def block(sd, pre, x, H, Wd, heads, ws, shift, mask, keep1=None, keep2=None):
    """swin_oracle.swin_block with the norms and gates whose parameters are there."""
    B, L, C = x.shape

    def branch(f, which, keep):
        if pre + f"post_norm{which}.weight" in sd:
            f = F.layer_norm(f, (C,), sd[pre + f"post_norm{which}.weight"], sd[pre + f"post_norm{which}.bias"])
        if pre + f"gate{which}" in sd:
            f = f * sd[pre + f"gate{which}"]
        return f if keep is None else f * keep.view(B, 1, 1).to(f.dtype)
    h = F.layer_norm(x, (C,), sd[pre + "norm1.weight"], sd[pre + "norm1.bias"]).view(B, H, Wd, C)
    He, We = max(H, ws), max(Wd, ws)
    h = F.pad(h, (0, 0, 0, We - Wd, 0, He - H))
    if shift > 0:
        h = torch.roll(h, (-shift, -shift), (1, 2))
    m = None if mask is None else mask.to(x.dtype)
    a = swin_oracle.window_attention(sd, pre + "attn.", swin_oracle._partition(h, ws), heads, ws, m)
    h = swin_oracle._unpartition(a, ws, He, We)
    if shift > 0:
        h = torch.roll(h, (shift, shift), (1, 2))
    x = x + branch(h[:, :H, :Wd, :].reshape(B, L, C), 1, keep1)
    y = F.layer_norm(x, (C,), sd[pre + "norm2.weight"], sd[pre + "norm2.bias"])
    y = F.linear(y, sd[pre + "mlp.0.weight"], sd[pre + "mlp.0.bias"])
    y = F.linear(F.gelu(y), sd[pre + "mlp.3.weight"], sd[pre + "mlp.3.bias"])
    return x + branch(y, 2, keep2)


OPTIONS = [dict(post_norm=True, layer_scale=0.5), dict(post_norm=True), dict(layer_scale=0.1)]


def build(dt, **options):
    from unet_amd.swin import SwinUNet
    cfg = dict(swin_oracle.DEFAULT_CONFIG, **options)
    m = SwinUNet(cfg, compute_dtype=dt)
    sd = W.fill_state_dict(swin_oracle.swin_template(cfg), seed=42)
    g = torch.Generator().manual_seed(7)
    for k, v in m.state_dict().items():
        if k not in sd:      # the added parameters: gates around their start, norms around one / zero
            base = cfg["layer_scale"] if "gate" in k else 1.0 if k.endswith("weight") else 0.0
            sd[k] = base + 0.2 * (base or 1.0) * torch.randn(v.shape, generator=g)
    m.load_state_dict(sd)
    return m.cuda(), sd, cfg


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("H,Wd", [(64, 64), (128, 64), (24, 24)])
def test_eval_forward(options, H, Wd, monkeypatch):
    monkeypatch.setattr(swin_oracle, "swin_block", block)
    x, _, _ = W.synthetic_batch(2, 4, H, Wd, seed=42)
    for dt, tol in ((torch.float32, 1e-4), (torch.bfloat16, 2e-2)):
        m, sd, cfg = build(dt, **options)
        out = m.eval()(x.cuda())
        ref, _ = swin_oracle.swin_unet_forward(sd, x, cfg, False)
        assert rel(out, ref) < tol, (dt, rel(out, ref))


@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("H,Wd", [(64, 64), (24, 24)])
def test_train_step_gradients(options, H, Wd, monkeypatch):
    monkeypatch.setattr(swin_oracle, "swin_block", block)
    x, y, _ = W.synthetic_batch(3, 4, H, Wd, seed=42)
    m, sd, cfg = build(torch.float32, **options)
    drop = [[torch.tensor([1.25, 0.0, 1.25]), torch.tensor([0.0, 1.25, 1.25])] if i % 2 else [None, None]
            for i in range(sum(cfg["depths"]))]
    m.train()
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
    names = list(leaves)
    num = sum(((got[k].grad.double().cpu() - leaves[k].grad) ** 2).sum() for k in names)
    den = sum((leaves[k].grad ** 2).sum() for k in names)
    assert (num / den).sqrt().item() < 2e-2
    for k in names:
        if "gate" in k or "post_norm" in k or ".norm" in k:
            if leaves[k].grad.norm() > 1e-7 * den.sqrt():
                assert rel(got[k].grad, leaves[k].grad) < 5e-2, k


def test_without_the_options_nothing_is_added():
    from unet_amd.swin import SwinUNet
    cfg = dict(swin_oracle.DEFAULT_CONFIG)
    assert list(SwinUNet(cfg).state_dict()) == list(swin_oracle.swin_template(cfg))


def test_gradient_sink_gets_every_gradient_once():
    x, _, _ = W.synthetic_batch(2, 4, 64, 64, seed=42)
    m, _, cfg = build(torch.bfloat16, **OPTIONS[0])
    m.train()
    m.drop_path_override = [[None, None]] * sum(cfg["depths"])
    m(x.cuda()).square().mean().backward()
    plain = {k: p.grad.clone() for k, p in m.named_parameters()}
    for p in m.parameters():
        p.grad = None
    seen = {}

    def sink(name, t):
        assert name not in seen
        seen[name] = t.clone()      # (on the stream that made it)
        return t
    m.grad_sink = sink
    m(x.cuda()).square().mean().backward()
    torch.cuda.synchronize()
    assert set(seen) == set(plain)
    for k in ("layers.0.blocks.1.norm1.weight", "layers.2.blocks.3.gate2", "layers.1.blocks.0.post_norm1.bias"):
        assert torch.equal(seen[k], plain[k]), k


def test_gated_step_in_a_graph_matches_the_eager_one():
    from oracle import loss_oracle
    from unet_amd import FusedAdamW, MultiLossFunction
    from unet_amd.graph import GraphedTrainStep
    crit = MultiLossFunction(loss_oracle.preset("weighted_mse_grad", grad_w=0.3, spec_w=0.0)).cuda()
    ref, got = (build(torch.float32, **OPTIONS[0])[0].train() for _ in range(2))
    for m in (ref, got):
        m.drop_path_override = [[None, None]] * 12
    opt_ref = FusedAdamW(ref.parameters(), lr=2e-3, weight_decay=0.05, max_grad_norm=1.0)
    opt_got = FusedAdamW(got.parameters(), lr=2e-3, weight_decay=0.05, max_grad_norm=1.0, capturable=True)
    g = torch.Generator().manual_seed(5)
    batches = [(torch.randn((2, 4, 64, 64), generator=g).cuda(), torch.randn((2, 1, 32, 32), generator=g).cuda(),
                torch.rand((2, 1, 32, 32), generator=g).cuda()) for _ in range(4)]
    step = GraphedTrainStep(got, crit, opt_got, *batches[0])
    for x, y, w in batches:
        opt_ref.zero_grad(set_to_none=True)
        loss, _ = crit(ref(x), y, w)
        loss.backward()
        opt_ref.step()
        replayed, _ = step(x, y, w)
        assert abs(replayed.item() - loss.item()) <= 1e-5 * max(1.0, abs(loss.item()))
    for (name, a), b in zip(ref.named_parameters(), got.parameters()):
        torch.testing.assert_close(b, a, rtol=1e-4, atol=2e-6, msg=name)


@pytest.mark.parametrize("options", [dict(), OPTIONS[0]])
@pytest.mark.parametrize("H,Wd", [(64, 64), (24, 24)])
def test_prediction_with_4_bit_linears(options, H, Wd, monkeypatch):
    """Every product of the pass against 64 bits on the inputs it really had (whole outputs are not comparable: where a
    chain is one rounding off, an activation's 4 bits turn over, and twelve blocks multiply that); and with the products
    replaced by unquantised ones the pass is the plain model's, so each stands where it should."""
    from unet_amd import ops
    x, _, _ = W.synthetic_batch(2, 4, H, Wd, seed=42)
    m, sd, cfg = build(torch.bfloat16, **options)
    m.eval()
    real, calls = ops.mx_linear, []
    weight = {}

    def checked(t, q, bias=None, act=0, resid=None, out=None, dtype=None):
        y = real(t, q, bias=bias, act=act, resid=resid, out=out, dtype=dtype)
        a, w = mx(t.float().cpu()).double().cuda(), mx(weight[id(q)].float().cpu()).double().cuda()
        want, mag = a @ w.t(), a.abs() @ w.abs().t()
        if bias is not None:
            want, mag = want + bias.double(), mag + bias.double().abs()
        if act == 2:
            want = want * 0.5 * torch.special.erfc(-want / 2 ** 0.5)
        if resid is not None:
            want, mag = want + resid.double(), mag + resid.double().abs()
        # fp32 sums of K <= 1536 terms, the GELU's 2.4e-7 of its argument, one rounding to bfloat16
        tol = (a.shape[-1] / 128 + 8) * 2.0 ** -24 * 1.13 * mag + 2.0 ** -21 * mag + 2.0 ** -8 * want.abs()
        bad = ((y.double() - want).abs() - tol).max().item()
        assert bad <= 0, (len(calls), act, resid is not None, bad)
        calls.append((act, resid is not None))
        return y

    def unquantised(t, q, bias=None, act=0, resid=None, out=None, dtype=None):
        y = F.linear(t.float(), weight[id(q)].float(), bias)
        y = F.gelu(y) if act == 2 else y
        return (y if resid is None else y + resid.float()).to(t.dtype)
    with torch.no_grad():
        plain = m(x.cuda())
        out = m.quantize_linears()(x.cuda())
        assert torch.equal(m(x.cuda()), out) and rel(out, plain) > 1e-3      # (they are in use)
        weight.update({id(q): w.detach() for w, q, _, _ in m._mx_linears})
        monkeypatch.setattr(ops, "mx_linear", checked)
        assert torch.equal(m(x.cuda()), out)
        assert len(calls) == 4 * 12 + 3 and sum(a == 2 for a, _ in calls) == 12
        monkeypatch.setattr(ops, "mx_linear", unquantised)
        assert rel(m(x.cuda()), plain) < 2e-2
        assert torch.equal(m.dequantize_linears()(x.cuda()), plain)


def test_changed_weights_are_refused_until_quantised_again():
    x, _, _ = W.synthetic_batch(1, 4, 64, 64, seed=42)
    m, sd, cfg = build(torch.bfloat16)
    m.eval().quantize_linears()
    with torch.no_grad():
        a = m(x.cuda())
        m.layers[1].blocks[0].mlp[0].weight.mul_(1.5)
        with pytest.raises(RuntimeError, match="quantize_linears"):
            m(x.cuda())
        b = m.quantize_linears()(x.cuda())
        assert not torch.equal(a, b)
    # training steps use the parameters
    m.train()
    m.drop_path_override = [[None, None]] * sum(cfg["depths"])
    t = m(x.cuda())
    m.dequantize_linears()
    assert torch.equal(m(x.cuda()), t)


def test_trained_weights_are_refused_until_quantised_again():
    """The optimizer's kernel writes the parameters without autograd's knowledge, and a captured step without Python's."""
    import unet_amd
    from unet_amd.graph import GraphedTrainStep
    x, y, _ = W.synthetic_batch(1, 4, 64, 64, seed=42)
    x, y = x.cuda(), y.cuda()
    m, _, _ = build(torch.bfloat16)

    def predict():
        m.eval()
        with torch.no_grad():
            return m(x)

    def loss(out, label):
        return ((out - F.interpolate(label, out.shape[-2:])) ** 2).mean()

    m.quantize_linears()
    a = predict()
    opt = unet_amd.FusedAdamW(m.parameters(), lr=1e-2, capturable=True)
    assert torch.equal(predict(), a)      # an optimizer alone changes nothing
    m.train()
    loss(m(x), y).backward()
    opt.step()
    with pytest.raises(RuntimeError, match="quantize_linears"):
        predict()
    m.quantize_linears()
    assert not torch.equal(predict(), a)
    m.train()
    step = GraphedTrainStep(m, loss, opt, x, y, warmup=2)
    m.quantize_linears()
    b = predict()
    m.train()
    for _ in range(2):
        step(x, y)
        with pytest.raises(RuntimeError, match="quantize_linears"):
            predict()
        m.quantize_linears()
        c = predict()
        assert not torch.equal(b, c)
        b = c


def test_one_block_of_operators_together():
    """The chain that a prediction runs: norm -> 4-bit product -> 4-bit product with GELU -> norm with gate and residual,
    against 64 bits on the operators' own intermediate values."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(3)
    C, M = 192, 640
    r = lambda *s, k=1.0: (torch.randn(*s, generator=g) * k)
    x = r(M, C).bfloat16().cuda()
    w1, w2 = r(4 * C, C, k=C ** -0.5).cuda(), r(C, 4 * C, k=(4 * C) ** -0.5).cuda()
    n1, n2, n3 = ((1 + 0.1 * r(C)).cuda() for _ in range(3))
    b = (0.1 * r(C)).cuda()
    q1, q2 = ops.mx_quantize(w1), ops.mx_quantize(w2)
    r0, ln, _ = ops.gated_norm_fwd(x, torch.zeros_like(x), pre=(n1, b), want_stats=False)
    assert torch.equal(r0, x)
    h = ops.mx_linear(ln, q1, act=2)
    f = ops.mx_linear(ops.mx_quantize(h), q2)
    r1, n, _ = ops.gated_norm_fwd(x, f, gate=n2, post=(n3, b), pre=(n1, None), kind="layer", want_stats=False)
    want_h = F.gelu(mx(ln.double().cpu()) @ mx(w1.double().cpu()).t())
    want_f = mx(h.double().cpu()) @ mx(w2.double().cpu()).t()
    post = F.layer_norm(f.double().cpu(), (C,), n3.double().cpu(), b.double().cpu())
    want_r = x.double().cpu() + n2.double().cpu() * post
    want_n = F.layer_norm(want_r, (C,), n1.double().cpu(), None)
    for got, want in ((h, want_h), (f, want_f), (r1, want_r), (n, want_n)):
        # one rounding to bfloat16, and fp32 sums of K <= 768 terms: (768 / 128 + 8) 2^-24 of magnitudes below 64
        tol = 2.0 ** -8 * want.abs() + 14 * 2.0 ** -24 * 64
        assert ((got.double().cpu() - want).abs() - tol).max() <= 0
