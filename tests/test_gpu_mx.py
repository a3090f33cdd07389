"""GPU tests of the microscaled 4-bit format (mx_quantize, mx_dequantize) and its product (mx_linear).

Quantisation is exact: the oracle below rounds in 64 bits and every value has to be equal.  The product's oracle is the
64-bit product of those values: E2M1 products are multiples of 1/4 up to 36 times two powers of two, and the sum over K is
taken in fp32, so a result is off by at most (K / 128 + 8) roundings of 2^-24 of the sum of magnitudes, and by one
rounding to bfloat16 (2^-8 of the value) where it is stored as such.  The GELU of the bfloat16 results is good to
1.5e-7 of its argument's size, which is below that.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def make(shape, seed, dt=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dt)


def quantised(x):
    """The values in 64 bits."""
    x = x.double().cpu()
    R, K = x.reshape(-1, x.shape[-1]).shape
    b = torch.zeros(R, (K + 31) // 32 * 32, dtype=torch.float64)
    b[:, :K] = x.reshape(R, K)
    b = b.view(R, -1, 32)
    big = b.abs().amax(-1, keepdim=True)
    e = torch.where((big > 0) & torch.isfinite(big), torch.frexp(torch.where(torch.isfinite(big), big, torch.ones_like(big)))[1] - 3, -127)
    scale = torch.pow(2.0, e.clamp(-127, 127).double())
    y = b / scale
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    q = (torch.round(y / step) * step).clamp(-6, 6) * scale
    q = torch.where(torch.isfinite(b).all(-1, keepdim=True), q, torch.full_like(q, float("nan")))
    return q.view(R, -1)[:, :K].reshape(x.shape)


def same(got, want):
    got, want = got.double().cpu(), want
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (5, 33), (64, 128), (65, 127), (63, 129), (100, 96), (17, 1001),
                                    (130, 384), (7, 4096), (300, 40)])
def test_round_trip(rows, K, dt):
    from unet_amd import ops
    x = (make((rows, K), rows + K) * torch.exp2(make((rows, K), 3) * 3)).to(dt)
    q = ops.mx_quantize(x.cuda())
    want = quantised(x)
    same(ops.mx_dequantize(q, F32), want)
    same(ops.mx_dequantize(q, BF), want)
    assert tuple(q.shape) == (rows, K)


def test_every_border_and_tie():
    """All midpoints between two codes, their neighbours in float32, both signs, under scales from 2^-120 to 2^120."""
    from unet_amd import ops
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.9999995])
    v = torch.cat([mids, torch.nextafter(mids, torch.zeros(1)), torch.nextafter(mids, torch.full((1,), 9.0)).clamp(max=7.9999995)])
    v = torch.cat([v, -v, torch.tensor([0.0, -0.0, 4.0, -4.0])])[None]      # 64 values; 4 fixes the scale at 1
    assert v.shape[1] == 64
    v = torch.cat([v[:, :28], torch.full((1, 4), 4.0), v[:, 28:56], torch.full((1, 4), 4.0), v[:, 56:], torch.full((1, 24), 4.0)], 1)
    rows = torch.cat([v * 2.0 ** e for e in range(-120, 121, 8)])
    same(ops.mx_dequantize(ops.mx_quantize(rows.cuda()), F32), quantised(rows))


def test_zeros_denormals_and_the_largest_numbers():
    from unet_amd import ops
    big, tiny = torch.finfo(F32).max, 2.0 ** -149
    x = torch.zeros(8, 64)
    x[1, 3], x[1, 40] = tiny, -tiny
    x[2, 0], x[2, 33] = big, -big
    x[3] = torch.linspace(-1, 1, 64) * 2.0 ** -126
    x[4] = torch.linspace(-1, 1, 64) * 2.0 ** -128
    x[5] = torch.linspace(-1, 1, 64) * 2.0 ** -125
    x[6, :32] = -0.0
    x[7] = torch.linspace(-1, 1, 64) * big
    same(ops.mx_dequantize(ops.mx_quantize(x.cuda()), F32), quantised(x))


def test_a_block_with_nan_or_infinity_is_nan_alone():
    from unet_amd import ops
    for dt in (F32, BF):
        x = make((70, 200), 5, dt)
        x[3, 40], x[69, 199], x[10, 0] = float("nan"), float("inf"), float("-inf")
        q = ops.mx_quantize(x.cuda())
        want = quantised(x)
        assert torch.isnan(want).sum() == 32 + 8 + 32
        same(ops.mx_dequantize(q, F32), want)
        w = make((130, 200), 6)
        y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda())).float().cpu()
        rows = torch.isnan(y).all(1)
        assert rows.nonzero().flatten().tolist() == [3, 10, 69] and not torch.isnan(y[~rows]).any()
        wn = w.clone()
        wn[7, 100] = float("nan")
        y = ops.mx_linear(make((70, 200), 7, dt).cuda(), ops.mx_quantize(wn.cuda())).float().cpu()
        cols = torch.isnan(y).all(0)
        assert cols.nonzero().flatten().tolist() == [7] and not torch.isnan(y[:, ~cols]).any()


def gelu(v):
    return v * 0.5 * torch.special.erfc(-v / 2 ** 0.5)


def check_linear(rows, K, N, dt, bias=True, act=0, resid=True, x=None, scale=1.0, seed=0):
    from unet_amd import ops
    x = (make((rows, K), seed + 1) * torch.exp2(make(K, seed + 2))).to(dt) if x is None else x
    w = make((N, K), seed + 3, F32, K ** -0.5 * scale)
    b = make(N, seed + 4) if bias else None
    r = make((rows, N), seed + 5, dt) if resid else None
    cu = lambda t: None if t is None else t.cuda()
    qw = ops.mx_quantize(w.cuda())
    got = ops.mx_linear(x if x.is_cuda else x.cuda(), qw, bias=cu(b), act=act, resid=cu(r))
    xv, wv = quantised(x).cuda(), quantised(w).cuda()
    want, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if b is not None:
        want, mag = want + b.cuda().double(), mag + b.cuda().double().abs()
    want = gelu(want) if act == 2 else want
    if r is not None:
        want, mag = want + r.cuda().double(), mag + r.cuda().double().abs()
    assert got.shape == (rows, N) and got.dtype == dt
    tol = (K / 128 + 8) * 2.0 ** -24 * (1.13 if act == 2 else 1.0) * mag + (2.0 ** -8 * want.abs() if dt == BF else 0.0)
    if act == 2:
        tol = tol + 2.0 ** -21 * mag      # the erf form: 1.5e-7 of the argument (bf16), a few roundings of erff (fp32)
    bad = ((got.double() - want).abs() - tol).max().item()
    assert bad <= 0, bad
    # an activation quantised beforehand gives the same bits
    pre = ops.mx_linear(ops.mx_quantize(x if x.is_cuda else x.cuda()), qw, bias=cu(b), act=act, resid=cu(r), dtype=dt)
    assert torch.equal(pre, got)
    return got


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("rows,K,N", [(1, 1, 1), (1, 32, 16), (1, 4096, 4096), (2, 129, 65), (15, 768, 40), (16, 128, 128), (17, 96, 384),
                                      (33, 200, 200), (64, 384, 96), (65, 1000, 333), (127, 31, 129), (128, 256, 256),
                                      (200, 2072, 1511), (513, 640, 136), (1037, 72, 30), (300, 8192, 64), (600, 1000, 700), (500, 64, 1100),
                                      (700, 1500, 1001), (20, 900, 24600), (30000, 900, 33), (64, 800, 25000), (4100, 5, 1)])
def test_product(rows, K, N, dt):
    check_linear(rows, K, N, dt)


@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("resid", [False, True])
def test_epilogues(act, bias, resid):
    for dt in (F32, BF):
        check_linear(70, 192, 72, dt, bias, act, resid)
        check_linear(5, 320, 100, dt, bias, act, resid)
        check_linear(3000, 96, 96, dt, bias, act, resid)


@pytest.mark.parametrize("rows,K,N", [(4096, 96, 288), (4096, 192, 768), (1024, 384, 1152), (256, 768, 2304), (256, 1536, 384),
                                      (2048, 2048, 2048), (8, 8192, 1024), (40000, 96, 96)])
def test_layer_shapes(rows, K, N):
    check_linear(rows, K, N, BF, act=2, resid=False)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("rows,K,N", [(3400, 900, 3100), (500, 100, 13000), (1000, 200, 10300), (900, 300, 10304), (1000, 400, 10300),
                                      (1000, 520, 10300), (3329, 1031, 3585)])
def test_large_products(rows, K, N, dt):
    """256 x 256 tiles: one to nine steps of K (the pipeline is four deep), ragged last tiles."""
    check_linear(rows, K, N, dt, act=2)
    check_linear(rows, K, N, dt, act=0, resid=False)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("K", [8, 100, 128, 136, 256, 300, 384, 500, 640, 700, 768])
def test_many_rows_of_every_step_count(K, dt):
    few = (K + 127) // 128 * 512
    check_linear(few + 65, K, 200, dt, act=2)
    check_linear(few, K, 77, dt, act=0, resid=False)
    check_linear(few - 1, K, 77, dt, act=0, resid=False)


def test_more_columns_than_a_workgroup_takes():
    check_linear(1030, 64, 9000, BF, resid=False)


@pytest.mark.parametrize("rows,K,N", [(1100, 200, 130), (1500, 700, 7000), (3400, 900, 3100), (20, 300, 40),
                                      (3200, 700, 130), (600, 1000, 700)])
def test_nan_stays_in_its_rows_and_columns(rows, K, N):
    from unet_amd import ops
    x, w = make((rows, K), 1, BF), make((N, K), 2)
    x[rows - 1, K - 1], x[5, 0] = float("nan"), float("inf")
    w[N - 1, 3] = float("-inf")
    y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda()), act=2).float().cpu()
    bad = torch.zeros(rows, N, dtype=torch.bool)
    bad[rows - 1], bad[5], bad[:, N - 1] = True, True, True
    assert torch.equal(torch.isnan(y), bad)


def test_products_are_exact_where_fp32_is():
    """Small whole numbers: every sum is exact, so the result is, whatever the order."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(0)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
    for rows, K, N in [(1, 256, 64), (9, 160, 70), (30, 512, 50), (100, 512, 260), (1700, 384, 400), (3400, 1152, 3100)]:
        x = grid[torch.randint(0, 8, (rows, K), generator=g)] * (torch.randint(0, 2, (rows, K), generator=g) * 2 - 1)
        w = grid[torch.randint(0, 8, (N, K), generator=g)] * (torch.randint(0, 2, (N, K), generator=g) * 2 - 1)
        x[:, ::32], w[:, ::32] = 4.0, 6.0      # every block's scale is 1
        y = ops.mx_linear(x.cuda(), ops.mx_quantize(w.cuda()))
        assert torch.equal(y.double().cpu(), x.double() @ w.double().t())


def test_scales_far_from_one():
    for s in (2.0 ** -100, 2.0 ** 60):
        check_linear(20, 256, 48, F32, bias=False, resid=False, scale=s)


def test_strided_operands_and_leading_dimensions():
    from unet_amd import ops
    for dt in (F32, BF):
        wide = make((2, 9, 3 * 96), 1, dt).cuda()
        w = make((40, 96), 2)
        qw = ops.mx_quantize(w.cuda())
        x = wide[..., 96:192]
        want = ops.mx_linear(x.contiguous(), qw)
        assert want.shape == (2, 9, 40)
        assert torch.equal(ops.mx_linear(x, qw), want)
        odd = make(18 * 97 + 1, 3, dt).cuda()[1:].view(18, 97)[:, 1:]
        assert torch.equal(ops.mx_linear(odd, qw), ops.mx_linear(odd.contiguous(), qw))
        for lo in (0, 8, 5):
            buf = torch.full((2, 9, 64), 7.0, dtype=dt, device="cuda")
            res = make((2, 9, 40), 4, dt).cuda()
            out = buf[..., lo:lo + 40]
            assert ops.mx_linear(x, qw, resid=res, out=out) is out
            assert torch.equal(out, ops.mx_linear(x, qw, resid=res))
            assert (buf[..., :lo] == 7).all() and (buf[..., lo + 40:] == 7).all()      # nothing else is written
            # in place on the residual
            acc = res.clone()
            ops.mx_linear(x, qw, resid=acc, out=acc)
            assert torch.equal(acc, out)


def test_no_rows_and_no_columns():
    from unet_amd import ops
    qw = ops.mx_quantize(make((40, 96), 1).cuda())
    x = torch.empty((0, 96), device="cuda")
    assert ops.mx_linear(x, qw).shape == (0, 40)
    assert ops.mx_dequantize(ops.mx_quantize(x)).shape == (0, 96)
    none = ops.mx_quantize(torch.empty((0, 96), device="cuda"))
    assert ops.mx_linear(torch.zeros((3, 96), device="cuda"), none).shape == (3, 0)


def test_other_stream_and_graph_replay():
    from unet_amd import ops
    qw = ops.mx_quantize(make((200, 384), 1).cuda())
    b = make(200, 2).cuda()
    for rows in (1, 50, 3000):
        x = make((rows, 384), 3, BF).cuda()
        run = lambda: ops.mx_linear(x, qw, bias=b, act=2)
        want = run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [run() for _ in range(2)]
        side.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], want)
        one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(one):
            o1 = run()
        with torch.cuda.graph(two):
            o2 = run()
        for k in range(4):
            x.copy_(make((rows, 384), 10 + k, BF).cuda())
            want = run()
            one.replay()
            two.replay()
            torch.cuda.synchronize()
            assert torch.equal(o1, want) and torch.equal(o2, want), (rows, k)


def test_refusals():
    from unet_amd import ops
    x, w = torch.zeros((4, 96), device="cuda"), torch.zeros((40, 96), device="cuda")
    qw = ops.mx_quantize(w)
    for f in (lambda: ops.mx_quantize(x.half()), lambda: ops.mx_quantize(x.t()), lambda: ops.mx_quantize(x[:, :0]),
              lambda: ops.mx_dequantize(qw, torch.float16), lambda: ops.mx_linear(x[:, :64], qw),
              lambda: ops.mx_linear(x, qw, bias=torch.zeros(39, device="cuda")), lambda: ops.mx_linear(x, qw, act=1),
              lambda: ops.mx_linear(x, qw, resid=torch.zeros((4, 39), device="cuda")),
              lambda: ops.mx_linear(x, qw, resid=torch.zeros((4, 40), device="cuda", dtype=BF)),
              lambda: ops.mx_linear(x, qw, out=torch.zeros((40, 4), device="cuda").t()),
              lambda: ops.mx_linear(x, qw, bias=torch.zeros(40)), lambda: ops.mx_linear(x, qw, dtype=BF),
              lambda: ops.mx_linear(x[:1].expand(4, 96), qw)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: ops.mx_linear(x, w), lambda: ops.mx_dequantize(x), lambda: ops.mx_linear([1.0], qw)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(RuntimeError):
        ops.mx_quantize(x.cpu())
    y = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.mx_linear(y, qw)
    with torch.no_grad():
        ops.mx_linear(y, qw)


def test_operands_that_share_memory():
    from unet_amd import ops
    for dt in (F32, BF):
        qw, qn = ops.mx_quantize(make((96, 96), 2).cuda()), ops.mx_quantize(make((40, 96), 2).cuda())
        wide = make((600, 200), 1, dt).cuda()
        x, want = wide[:, :96], ops.mx_linear(wide[:, :96].contiguous(), qw)
        assert torch.equal(ops.mx_linear(x, qw, out=wide[:, 96:192]), want)      # beside each other in one buffer
        r = make((600, 40), 5, dt).cuda()
        for out in (x, wide[:, 8:104], wide[:, 95:191]):
            with pytest.raises(ValueError, match="shares memory with x"):
                ops.mx_linear(x, qw, out=out)
        buf = make((600, 64), 3, dt).cuda()
        with pytest.raises(ValueError, match="without being resid"):
            ops.mx_linear(x, qn, resid=buf[:, :40], out=buf[:, 8:48])
        with pytest.raises(ValueError, match="without being resid"):
            ops.mx_linear(x[1:], qn, resid=r[1:], out=r[:-1])
        want = ops.mx_linear(x, qn, resid=r)
        assert torch.equal(ops.mx_linear(x, qn, resid=r, out=r), want)


def test_rows_beyond_32_bits():
    """A wide row stride puts the last rows past 2^32 bytes, on either side."""
    from unet_amd import ops
    qw = ops.mx_quantize(make((72, 96), 2).cuda())
    for rows, ld in ((20, 1 << 27), (600, 1 << 22)):
        big = torch.empty(rows * ld, dtype=BF, device="cuda").view(rows, ld)
        x = make((rows, 96), 1, BF).cuda()
        big[:, :96] = x
        want = ops.mx_linear(x, qw)
        assert torch.equal(ops.mx_linear(big[:, :96], qw), want)
        assert torch.equal(ops.mx_quantize(big[:, :96]).data, ops.mx_quantize(x).data)
        big[:, 200:300] = 7
        ops.mx_linear(x, qw, out=big[:, 208:280])
        assert torch.equal(big[:, 208:280], want) and (big[:, 200:208] == 7).all() and (big[:, 280:300] == 7).all()
        del big
