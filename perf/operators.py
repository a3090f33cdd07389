"""The token-block operators as a benchmark calls them: gated norms (norm behind a branch, gate, residual scale, norm in
front of the next branch; forward and backward) and microscaled 4-bit products.

``run`` computes a case in elementary torch operations, or, with ``own`` set, through ``unet_amd.ops``.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # magnitudes of the 4-bit format E2M1


# ------------------------------------------------------------------ the cases
def _norm(name, rows, width, dtype, kind="layer", post=True, gate=True, pre=True, samples=0, scale=1.0, train=False):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "kind": kind, "post": post,
            "gate": gate, "pre": pre, "samples": samples, "scale": scale, "train": train}


def _linear(name, rows, k, n, dtype, bias=True, act=0, resid=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias, "act": act,
            "resid": resid}


def _store(name, rows, k, dtype):
    return {"name": name, "op": "store", "rows": rows, "k": k, "dtype": dtype}


def listed():
    return [
        # one 256-pixel patch at the deepest Swin stage (8 x 8 tokens of 768 channels): the smallest call, latency
        _norm("norm_one_patch", 64, 768, "bf16"),
        # prediction of 64 patches at the first stage (64 x 64 tokens of 96 channels): the widest token grid
        _norm("norm_predict_stage0", 64 * 4096, 96, "bf16"),
        # training step of 64 patches at the second stage, DropPath factors per sample
        _norm("norm_train_stage1", 64 * 1024, 192, "bf16", samples=64, train=True),
        # a wide token model in training: RMS norm in front, gated branch without a norm behind it, scaled residual
        _norm("norm_train_wide_rms", 8192, 4096, "bf16", kind="rms", post=False, scale=0.75, train=True),
        # float32 training, a width and a row count that divide by nothing
        _norm("norm_train_odd_f32", 5003, 1001, "f32", train=True),
        # a tensor kept in 4 bits and read back: the hidden activations of the second stage
        _store("store_hidden", 64 * 1024, 768, "bf16"),
        # the same for a small float32 matrix whose last block of 32 is short
        _store("store_odd_f32", 77, 1001, "f32"),
        # a single token through a square layer: the weights are all there is to read
        _linear("linear_token", 1, 4096, 4096, "bf16"),
        # fc1 with GELU at the first Swin stage, 64 patches
        _linear("linear_stage0_fc1", 64 * 4096, 96, 384, "bf16", act=2),
        # qkv at the third Swin stage, 64 patches
        _linear("linear_stage2_qkv", 64 * 256, 384, 1152, "bf16"),
        # float32 activations, residual, sizes that divide by nothing
        _linear("linear_odd_f32", 1037, 2072, 1511, "f32", resid=True),
        # a large square product
        _linear("linear_large", 8192, 8192, 8192, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the widths of token stages and wide models, from one row to a few hundred thousand, every third
    size rounded to a multiple of 32 as real layers are, the others left as they fall."""
    def size(lo, hi):
        v = _log(rng, lo, hi)
        return max(32, v // 32 * 32) if rng.random() < 0.34 else v
    dt = rng.choice(["bf16", "bf16", "f32"])
    op = rng.choice(["norm", "norm", "linear", "linear", "store"])
    if op == "linear":
        k, n = size(32, 8192), size(32, 8192)
        rows = _log(rng, 1, max(16, min(1 << 17, (1 << 38) // (k * n), (1 << 26) // max(k, n))))
        c = _linear("", rows, k, n, dt, rng.random() < 0.8, rng.choice([0, 0, 2]), rng.random() < 0.4)
    elif op == "store":
        k = size(32, 8192)
        c = _store("", _log(rng, 1, (1 << 25) // k), k, dt)
    else:
        width = size(32, 8192)
        samples = rng.choice([0, 1, 4, 16])
        rows = _log(rng, 1, (1 << (25 if dt == "bf16" else 24)) // width)
        if samples:
            rows = max(1, rows // samples) * samples
        post, gate = rng.random() < 0.6, rng.random() < 0.7
        c = _norm("", rows, width, dt, rng.choice(["layer", "layer", "rms"]), post, gate, rng.random() < 0.85, samples,
                  rng.choice([1.0, 0.75, 1.4142135]), rng.random() < 0.6)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, to=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(mean).to(to)
    s = {"case": dict(case)}
    if case["op"] == "norm":
        M, C = case["rows"], case["width"]
        s["x"] = normal(M, C, scale=1.5, mean=0.1, to=dt)
        s["f"] = normal(M, C, scale=0.6, mean=-0.05, to=dt)
        bias = case["kind"] == "layer"
        s["post"] = (normal(C, scale=0.1, mean=1.0), normal(C, scale=0.1) if bias else None) if case["post"] else None
        s["pre"] = (normal(C, scale=0.1, mean=1.0), normal(C, scale=0.1) if bias else None) if case["pre"] else None
        s["gate"] = normal(C, scale=0.2, mean=0.5) if case["gate"] else None
        s["keep"] = None
        if case["samples"]:     # DropPath factors: 0 or 1 / (1 - p)
            u = torch.rand(case["samples"], generator=g, device="cuda")
            s["keep"] = (u < 0.9).float() / 0.9
        if case["train"]:
            s["dr"] = normal(M, C, scale=0.02, to=dt)
            s["dn"] = normal(M, C, scale=0.02, to=dt) if case["pre"] else None
        return s
    if case["op"] == "store":
        x = normal(case["rows"], case["k"])
        # activations: channels of very different size
        s["x"] = (x * torch.exp2(torch.randn(case["k"], generator=g, device="cuda"))).to(dt)
        return s
    M, K, N = case["rows"], case["k"], case["n"]
    s["x"] = (normal(M, K) * torch.exp2(0.5 * torch.randn(K, generator=g, device="cuda"))).to(dt)
    w = normal(N, K, scale=K ** -0.5)
    s["bias"] = normal(N, scale=0.1) if case["bias"] else None
    s["resid"] = normal(M, N, to=dt) if case["resid"] else None
    if own:
        from unet_amd import ops
        s["w"] = ops.mx_quantize(w)
    else:
        codes, exps = _quantize(w)
        s["w"] = (codes[:, 0::2] | codes[:, 1::2] << 4, exps)      # two codes a byte, as the weights are kept
    return s


# ------------------------------------------------------------------ plain forms
def _blocks(x):
    """(rows, ceil(K / 32), 32), the last block filled with zeros."""
    R, K = x.shape
    pad = -K % 32
    if pad:
        x = torch.cat([x, x.new_zeros(R, pad)], 1)
    return x.view(R, -1, 32)


def _quantize(x):
    """E2M1 codes (rows, padded K) and the exponents of the blocks' scales (rows, blocks); exponent 128: not a number."""
    b = _blocks(x.float())
    big = b.abs().amax(-1)
    se = (torch.frexp(big)[1] - 3).clamp(-127, 127)
    se = torch.where(big > 0, se, torch.full_like(se, -127))
    # in 64 bits: division by the power of two is exact, and so is every comparison with a border between two codes
    inv = ((1023 - se.long()) << 52).view(torch.float64)
    a = b.double().abs() * inv.unsqueeze(-1)
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() +
            (a >= 3.5).byte() + (a > 5.0).byte())
    code = code | (torch.signbit(b).byte() << 3)
    bad = ~torch.isfinite(b).all(-1)
    se = torch.where(bad, torch.full_like(se, 128), se)
    return code.view(x.shape[0], -1), se


def _values(codes, exps, K):
    """float32 values of codes and block exponents."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=codes.device)
    v = grid[codes.int()].view(codes.shape[0], -1, 32)
    scale = ((1023 + exps.long()) << 52).view(torch.float64).float()
    scale = torch.where(exps == 128, torch.full_like(scale, float("nan")), scale)
    return (v * scale.unsqueeze(-1)).view(codes.shape[0], -1)[:, :K]


def _gelu(v):
    return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))


def _plain_linear(s):
    case, x = s["case"], s["x"]
    K = case["k"]
    packed, exps = s["w"]
    codes = torch.stack([packed & 15, packed >> 4], -1).view(packed.shape[0], -1)
    w = _values(codes, exps, K)
    y = _values(*_quantize(x), K) @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == 2:
        y = _gelu(y)
    if s["resid"] is not None:
        y = y + s["resid"].float()
    return y.to(x.dtype)


def _moments(v, kind):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    d = v - mean
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + _EPS)
    return d * rstd, rstd


def _affine(hat, p):
    y = hat * p[0]
    return y if p[1] is None else y + p[1]


def _col(v):
    """Sum over the rows: a long sum, in 64 bits."""
    return v.double().sum(0).float()


def _norm_grad(g, hat, rstd, kind):
    m = g.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (g - m - hat * (g * hat).mean(-1, keepdim=True))


def _plain_norm(s):
    case, kind = s["case"], s["case"]["kind"]
    dt = s["x"].dtype
    x, f = s["x"].float(), s["f"].float()
    M = x.shape[0]
    keep = None if s["keep"] is None else s["keep"].repeat_interleave(M // s["keep"].numel()).unsqueeze(1)
    h = f
    if s["post"] is not None:
        fhat, frstd = _moments(f, kind)
        h = _affine(fhat, s["post"])
    b = h if s["gate"] is None else h * s["gate"]
    if keep is not None:
        b = b * keep
    r = x * case["scale"] + b
    out = [r.to(dt)]
    if s["pre"] is not None:
        rhat, rrstd = _moments(r, kind)
        out.append(_affine(rhat, s["pre"]).to(dt))
    if not case["train"]:
        return out
    g = s["dr"].float()
    grads = []
    if s["pre"] is not None:
        dn = s["dn"].float()
        g = g + _norm_grad(dn * s["pre"][0], rhat, rrstd, kind)
        grads += [_col(dn * rhat)] + ([] if s["pre"][1] is None else [_col(dn)])
    u = g if keep is None else g * keep
    dh = u
    if s["gate"] is not None:
        grads.append(_col(u * h))
        dh = u * s["gate"]
    df = dh
    if s["post"] is not None:
        df = _norm_grad(dh * s["post"][0], fhat, frstd, kind)
        grads += [_col(dh * fhat)] + ([] if s["post"][1] is None else [_col(dh)])
    return out + [(g * case["scale"]).to(dt), df.to(dt)] + grads


# ------------------------------------------------------------------ one pass
def _own(s):
    from unet_amd import ops
    case = s["case"]
    if case["op"] == "linear":
        return ops.mx_linear(s["x"], s["w"], bias=s["bias"], act=case["act"], resid=s["resid"])
    if case["op"] == "store":
        return ops.mx_dequantize(ops.mx_quantize(s["x"]), s["x"].dtype)
    kw = dict(gate=s["gate"], keep=s["keep"], res_scale=case["scale"], post=s["post"], pre=s["pre"], kind=case["kind"],
              eps=_EPS)
    r, n, stats = ops.gated_norm_fwd(s["x"], s["f"], want_stats=case["train"], **kw)
    out = [r] if n is None else [r, n]
    if not case["train"]:
        return out
    d = ops.gated_norm_bwd(s["dr"], s["dn"], s["x"], s["f"], stats, **kw)
    grads = [d.pre_weight, d.pre_bias, d.gate, d.post_weight, d.post_bias]
    return out + [d.x, d.f] + [t for t in grads if t is not None]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "linear":
        return _plain_linear(state)
    if op == "store":
        x = state["x"]
        return _values(*_quantize(x), x.shape[1]).to(x.dtype)
    return _plain_norm(state)


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        M, K, N = case["rows"], case["k"], case["n"]
        kb = -(-K // 32)
        b = M * K * e + N * (K // 2 + kb) + M * N * e * (2 if case["resid"] else 1) + (4 * N if case["bias"] else 0)
        return {"bytes": b, "flops": 2 * M * K * N}
    if case["op"] == "store":
        M, K = case["rows"], case["k"]
        stored = M * (-(-K // 2) + -(-K // 32))
        return {"bytes": 2 * M * K * e + 2 * stored, "flops": 4 * M * K}
    M, C = case["rows"], case["width"]
    norms = int(case["post"]) + int(case["pre"])
    tensors, flops = 3 + int(case["pre"]), 4 + 8 * norms
    if case["train"]:
        # the forward pass, then the backward pass over x, f, dr, dn into dx, df
        tensors += 5 + int(case["pre"])
        flops += 8 + 14 * norms
    vectors = (2 if case["kind"] == "layer" else 1) * norms + int(case["gate"])
    return {"bytes": tensors * M * C * e + vectors * C * 4 * (3 if case["train"] else 1), "flops": flops * M * C}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_values(x):
    """Each block of 32 over 2^(floor(log2 max) - 2), rounded half to even to E2M1's steps, held to 6."""
    b = _blocks(x.double())
    e = torch.frexp(b.abs().amax(-1, keepdim=True))[1].double() - 3.0
    scale = torch.pow(torch.full_like(e, 2.0), e.clamp(-127, 127))
    y = b / scale
    octave = torch.frexp(y.abs().clamp_min(1.0))[1].double() - 1.0       # 0 below 2, 1 below 4, 2 below 8
    step = torch.pow(torch.full_like(octave, 2.0), octave - 1.0)
    y = (torch.round(y / step) * step).clamp(-6.0, 6.0)
    return (y * scale).view(x.shape[0], -1)[:, :x.shape[1]]


def _exact_norm(case, seed):
    s = prepare(case, seed)
    leaves = {}

    def leaf(name, t):
        if t is None:
            return None
        leaves[name] = t.double().requires_grad_(case["train"])
        return leaves[name]

    def normed(v, p):
        if case["kind"] == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS) * p[0]
        return v if p[1] is None else v + p[1]
    x, f = leaf("x", s["x"]), leaf("f", s["f"])
    pre = s["pre"] and (leaf("pw", s["pre"][0]), leaf("pb", s["pre"][1]))
    gate = leaf("g", s["gate"])
    post = s["post"] and (leaf("qw", s["post"][0]), leaf("qb", s["post"][1]))
    h = normed(f, post) if post else f
    if gate is not None:
        h = h * gate
    if s["keep"] is not None:
        S = s["keep"].numel()
        h = (h.view(S, -1) * s["keep"].double().unsqueeze(1)).view(h.shape)
    r = case["scale"] * x + h
    n = normed(r, pre) if pre else None
    out = [r.detach()] + ([] if n is None else [n.detach()])
    if not case["train"]:
        return out
    total = (r * s["dr"].double()).sum()
    if n is not None:
        total = total + (n * s["dn"].double()).sum()
    return out + list(torch.autograd.grad(total, list(leaves.values())))


def exact(case, seed):
    if case["op"] == "norm":
        return _exact_norm(case, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_values(s["x"])
    # the weights again, as prepare drew them: x's two draws, then the weights
    torch.randn(case["rows"], case["k"], generator=g, device="cuda")
    torch.randn(case["k"], generator=g, device="cuda")
    w = torch.randn(case["n"], case["k"], generator=g, device="cuda").mul_(case["k"] ** -0.5)
    y = _exact_values(s["x"]) @ _exact_values(w).t()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if case["act"] == 2:
        y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2.0))
    return y if s["resid"] is None else y + s["resid"].double()
