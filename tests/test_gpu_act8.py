"""Activation checkpoints in 8 bits against their definition in 64 bits.

Codes and steps are whole numbers and have to be equal. Sums are fp32: an
element of a weight gradient may be off by 2^-23 (64 + T / 256) sum_t |g v| --
each of the sixteen 16-token products of a 256-token stretch may lose up to
two units in the last place of the running sum on the tensor cores, and the
stretches are added one by one in fp32.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _pkg():
    import sae_b200
    return sae_b200


def held8(x):
    """(codes, step bytes, values float64) of a float64 [T, D] array."""
    T, D = x.shape
    ng = -(-D // 32)
    v = np.zeros((T, ng * 32))
    v[:, :D] = x
    v = v.reshape(T, ng, 32)
    amax = np.abs(v).max(2)
    bad = ~np.isfinite(v).all(2)
    safe = np.where(bad | (amax == 0), 1.0, amax)
    k = np.floor(np.log2(safe)).astype(int) - 6
    k = np.where(np.ldexp(safe, -k) >= 127.5, k + 1, k)
    k = np.where(np.ldexp(safe, 1 - k) < 127.5, k - 1, k)
    k = np.where(amax == 0, -126, np.maximum(k, -126))
    with np.errstate(invalid="ignore"):
        c = np.rint(np.ldexp(np.where(bad[:, :, None], 0.0, v), -k[:, :, None]))
    c = np.where((k >= 122)[:, :, None], np.clip(c, -63, 63), c)
    val = np.where(bad[:, :, None], np.nan, np.ldexp(c, k[:, :, None]))
    step = np.where(bad, 255, k + 127)
    return c.reshape(T, -1), step, val.reshape(T, -1)[:, :D]


def _check_held(x):
    B = _pkg()
    a = B.checkpoint8(x)
    codes, steps, val = held8(x.detach().reshape(-1, x.shape[-1]).double().cpu().numpy())
    assert np.array_equal(a.codes.cpu().numpy(), codes)
    assert np.array_equal(a.steps.cpu().numpy(), steps)
    for dt in (torch.float32, torch.bfloat16):
        got = a.dequantize(dt)
        assert got.shape == x.shape and got.dtype == dt
        np.testing.assert_array_equal(got.double().cpu().numpy().reshape(val.shape), val)
    return a


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,D", [(1, 1), (1, 32), (3, 33), (7, 31), (5, 777), (2, 40), (300, 1536),
                                 (1025, 64)])
def test_codes_are_the_definitions(T, D, dtype):
    g = torch.Generator(device=DEV).manual_seed(T * 1000 + D)
    x = torch.randn(T, D, device=DEV, generator=g) * torch.exp(
        4 * torch.randn(T, 1, device=DEV, generator=g))
    _check_held(x.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_at_the_borders(dtype):
    x = torch.zeros(12, 70)
    x[0, :] = 0.0
    x[1, 3] = 127.5                      # the next step up, exactly at the border
    x[2, 3] = 127.0
    x[3, :5] = torch.tensor([127.0, 0.5, 1.5, -0.5, 2.5])    # ties to even
    x[4, 2] = float("inf")               # only its own group is lost
    x[4, 40] = 3.0
    x[5, 69] = float("nan")
    x[6, 1] = 2.0 ** -130                # subnormal
    x[7, 33] = 2.0 ** -149
    x[8, 0] = torch.finfo(dtype).max     # the largest step saturates
    x[9, 0], x[9, 1] = 1.0, -torch.finfo(torch.float32).tiny
    x[10, 5] = 2.0 ** -119
    x[11, 64] = -1.9921875
    _check_held(x.to(dtype).to(DEV))


def test_leading_dimensions_strides_and_empty():
    B = _pkg()
    x = torch.randn(4, 6, 48, device=DEV)
    _check_held(x)
    wide = torch.randn(9, 200, device=DEV)
    _check_held(wide[:, 3:103])                 # rows apart, base not 16-byte aligned
    _check_held(wide[::2, :64])
    _check_held(wide.t())                       # columns apart: copied
    _check_held(torch.randn(1, 50, device=DEV).expand(5, 50))
    e = B.checkpoint8(torch.randn(0, 40, device=DEV))
    assert e.dequantize().shape == (0, 40)
    assert torch.equal(e.weight_grad(torch.randn(0, 7, device=DEV)), torch.zeros(7, 40, device=DEV))
    acc = torch.ones(7, 40, device=DEV)
    e.weight_grad(torch.randn(0, 7, device=DEV), out=acc, accumulate=True)
    assert torch.equal(acc, torch.ones(7, 40, device=DEV))
    a = B.checkpoint8(wide)
    out = torch.full((9, 301), 7.0, device=DEV)
    a.dequantize(out=out[:, 5:205])
    assert torch.equal(out[:, 5:205], a.dequantize())
    assert bool((out[:, :5] == 7).all()) and bool((out[:, 205:] == 7).all())


def _wgrad_bound(g, v, T):
    s = np.abs(g).T @ np.abs(v)
    return 2.0 ** -23 * (64 + T / 256) * s + 1e-37


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("gdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D,N", [(1, 1, 1), (1, 96, 256), (17, 33, 40), (64, 128, 256),
                                   (65, 130, 264), (300, 257, 515), (2050, 200, 301),
                                   (1000, 64, 2048)])
def test_weight_grad(T, D, N, gdtype, transposed):
    B = _pkg()
    gen = torch.Generator(device=DEV).manual_seed(T + D + N)
    x = torch.randn(T, D, device=DEV, generator=gen)
    g = (torch.randn(T, N, device=DEV, generator=gen) * 1e-3).to(gdtype)
    a = B.checkpoint8(x)
    got = a.weight_grad(g, transposed=transposed)
    assert got.shape == ((D, N) if transposed else (N, D)) and got.dtype == torch.float32
    _, _, v = held8(x.double().cpu().numpy())
    g64 = g.double().cpu().numpy()
    want, bound = g64.T @ v, _wgrad_bound(g64, v, T)
    got64 = got.double().cpu().numpy()
    assert (np.abs((got64.T if transposed else got64) - want) <= bound).all()
    # the same call gives the same bits; accumulate adds to what is there
    again = a.weight_grad(g, transposed=transposed)
    assert torch.equal(got, again)
    base = torch.randn(got.shape, device=DEV, generator=gen) * 1e-2
    acc = a.weight_grad(g, transposed=transposed, out=base.clone(), accumulate=True)
    off = (acc.double() - base.double()).cpu().numpy()
    off = off.T if transposed else off
    room = bound + 2.0 ** -23 * np.abs(acc.double().cpu().numpy().T if transposed
                                       else acc.double().cpu().numpy())
    assert (np.abs(off - want) <= room).all()


@pytest.mark.parametrize("T,D,N,gdtype", [(4096, 8192, 1024, torch.bfloat16),
                                         (2048, 20000, 512, torch.bfloat16),
                                         (1000, 49152, 264, torch.bfloat16),
                                         (4096, 16384, 512, torch.float32),
                                         (1000, 1536, 16384, torch.float32)])
@pytest.mark.parametrize("transposed", [False, True])
def test_weight_grad_of_more_tiles_than_pairs_of_sms(T, D, N, gdtype, transposed):
    """A pair of SMs goes on to a second tile while the first is still being stored
    (slowest when transposed): every call gives the same bits, within the bound."""
    B = _pkg()
    gen = torch.Generator(device=DEV).manual_seed(T + D + N)
    x = torch.randn(T, D, device=DEV, generator=gen).bfloat16()
    g = (torch.randn(T, N, device=DEV, generator=gen) * 1e-3).to(gdtype)
    a = B.checkpoint8(x)
    v, g64 = a.dequantize(torch.float32).double(), g.double()
    want, bound = g64.t() @ v, 2.0 ** -23 * (64 + T / 256) * (g64.abs().t() @ v.abs()) + 1e-37
    del v, g64
    other = torch.empty(256 << 20, device=DEV, dtype=torch.uint8)
    first = None
    for _ in range(5):
        other.zero_()                    # the operands leave the L2 cache
        got = a.weight_grad(g, transposed=transposed)
        first = got if first is None else first
        assert torch.equal(got, first)
    got = first.t() if transposed else first
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("gdtype", [torch.bfloat16, torch.float32])
def test_weight_grad_strides_and_rows_behind(gdtype):
    B = _pkg()
    T, D, N = 90, 96, 200
    x = torch.randn(T, D, device=DEV)
    gw = torch.randn(T, 400, device=DEV).to(gdtype)
    g = gw[:, 3:3 + N]                               # odd offset, rows apart
    a = B.checkpoint8(x)
    want = a.weight_grad(g.contiguous())
    out = torch.full((N + 3, D + 9), 5.0, device=DEV)
    a.weight_grad(g, out=out[2:2 + N, 4:4 + D])
    # both go through the same sums, whatever the strides
    np.testing.assert_allclose(out[2:2 + N, 4:4 + D].cpu(), want.cpu(), rtol=0, atol=float(
        2.0 ** -22 * 128 * (g.float().abs().t() @ a.dequantize().abs()).max()))
    out[2:2 + N, 4:4 + D] = 5.0
    assert bool((out == 5.0).all())
    b = B.checkpoint8(x.reshape(9, 10, D))
    assert torch.equal(b.weight_grad(g.contiguous().reshape(9, 10, N)), want)


def test_weight_grad_non_finite_group_stays_in_its_column():
    B = _pkg()
    x = torch.randn(200, 96, device=DEV)
    x[7, 40] = float("inf")
    g = torch.randn(200, 130, device=DEV).bfloat16()
    got = B.checkpoint8(x).weight_grad(g)
    assert bool(got[:, 32:64].isnan().all())
    assert bool(got[:, :32].isfinite().all()) and bool(got[:, 64:].isfinite().all())


@pytest.mark.parametrize("T,D,N,gdtype", [(6000, 40, 30000, torch.float32),   # parts of g in two
                                          (2100, 33000, 1100, torch.bfloat16)])  # values in two
def test_weight_grad_of_more_tokens_than_one_launch_takes(T, D, N, gdtype):
    B = _pkg()
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(T, D, device=DEV, generator=gen)
    g = torch.randn(T, N, device=DEV, generator=gen).to(gdtype)
    a = B.checkpoint8(x)
    v = a.dequantize(torch.float32).double()
    base = torch.randn(N, D, device=DEV, generator=gen)
    got = a.weight_grad(g, out=base.clone(), accumulate=True).double()
    want = g.double().t() @ v
    size = g.double().abs().t() @ v.abs()
    bound = 2.0 ** -23 * (64 + T / 256) * size + 2.0 ** -22 * (got.abs() + base.double().abs())
    assert bool(((got - base.double() - want).abs() <= bound).all())


def _jump_inputs(T, F, dtype, eps, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    log_thr = (-2.3 + 0.3 * torch.randn(F, device=DEV, generator=g))
    theta = log_thr.double().exp()
    pre = (0.4 * torch.randn(T, F, device=DEV, generator=g) - 0.1).to(dtype)
    at = (pre.double() - theta) * (126 / eps)
    pre[((at - at.round()).abs() < 1e-3) & (at.abs() < 127)] = -3.0   # clear of the codes' borders
    return pre, log_thr, theta


@pytest.mark.parametrize("gate_kind", ["scalar", "full", "row", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,F", [(1, 1), (1, 1000), (3, 17), (64, 128), (65, 1028), (517, 301)])
def test_jumprelu8(T, F, dtype, gate_kind):
    B = _pkg()
    eps = 0.1875
    pre, log_thr, theta = _jump_inputs(T, F, dtype, eps, T + F)
    gen = torch.Generator(device=DEV).manual_seed(5)
    gf = torch.randn(T, F, device=DEV, generator=gen) * 1e-3
    gg = {"scalar": torch.randn(1, 1, device=DEV, generator=gen).expand(T, F),
          "row": torch.randn(T, 1, device=DEV, generator=gen).expand(T, F),
          "full": torch.randn(T, F, device=DEV, generator=gen), "none": None}[gate_kind]
    pre.requires_grad_()
    log_thr.requires_grad_()
    feat, gate = B.jumprelu8(pre, log_thr, eps)
    p64, u = pre.detach().double(), pre.detach().double() - theta
    on, band = u > 0, u.abs() < eps
    assert torch.equal(gate, on.float()) and torch.equal(feat, pre.detach().float() * on)
    outs, seeds = ((feat, gate), (gf, gg)) if gg is not None else ((feat,), (gf,))
    gp, gt = torch.autograd.grad(outs, (pre, log_thr), seeds)
    assert gp.dtype == dtype and torch.equal(gp, (gf * on).to(dtype))
    held = theta + (torch.ceil(u * 126 / eps) - 0.5) * eps / 126
    assert float(((held - p64).abs() * band).max()) <= eps / 252 * (1 + 1e-12)
    term = torch.where(band, held * gf.double() + (0 if gg is None else gg.double()), 0.0)
    # theta + (code - 1/2) step cancels where the value is near zero: theta's rounding (expf, 2
    # ulp), the step's and the sum's are relative to theta + eps, not to the value.
    size = torch.where(band, ((theta + eps) * gf.double()).abs()
                       + (0 if gg is None else gg.double().abs()), 0.0)
    want = -term.sum(0) * theta / (2 * eps)
    # 64 tokens are added in fp32, then 8 half-ulps for the value, its product and the result
    bound = 2.0 ** -24 * (64 + 8) * size.sum(0) * theta / (2 * eps) + 1e-37
    assert bool(((gt.double() - want).abs() <= bound).all())


def test_jumprelu8_masked_places_are_not_read():
    """Infinities and NaN where the gate is closed reach neither gradient."""
    B = _pkg()
    T, F, eps = 70, 64, 0.125
    pre, log_thr, theta = _jump_inputs(T, F, torch.float32, eps, 3)
    pre[5, 7] = float("-inf")
    pre[6, 8] = float("inf")
    pre[6, 9] = float("nan")
    off = pre.double() - theta < -eps
    gf = torch.where(off, torch.tensor(float("nan"), device=DEV), torch.ones(T, F, device=DEV))
    gf[6, 9] = float("inf")
    pre.requires_grad_()
    log_thr.requires_grad_()
    feat, gate = B.jumprelu8(pre, log_thr, eps)
    f, on = feat.detach(), gate.detach()
    assert float(f[5, 7]) == 0.0 and float(f[6, 8]) == float("inf")
    assert bool(f[6, 9].isnan()) and float(on[6, 9]) == 0.0
    gp, gt = torch.autograd.grad((feat, gate), (pre, log_thr), (gf, gf))
    assert bool((gp[off] == 0).all()) and float(gp[6, 9]) == 0.0 and float(gp[6, 8]) == 1.0
    assert bool(gt.isfinite().all())


def test_jumprelu8_difference_and_partial_gradients():
    """grad_pre against a difference of the loss where no gate opens or closes;
    each output's gradient alone; a leading dimension; no tokens."""
    B = _pkg()
    eps = 0.125
    pre, log_thr, theta = _jump_inputs(12, 96, torch.float32, eps, 9)
    w = torch.randn(12, 96, device=DEV)
    p = pre.clone().requires_grad_()
    t = log_thr.clone().requires_grad_()
    (B.jumprelu8(p, t, eps)[0] * w).sum().backward()
    clear = (pre.double() - theta).abs() > 2e-3
    up = (B.jumprelu8(pre + 1e-3, log_thr, eps)[0] - B.jumprelu8(pre - 1e-3, log_thr, eps)[0]) * w
    # feat is linear there: only the rounding of pre +- 1e-3 and of the quotient is left
    scale = pre.abs() + 1e-3
    assert bool((((up / 2e-3 - p.grad).abs() <= 2.0 ** -22 * scale * w.abs() / 1e-3 + 2.0 ** -22)
                 | ~clear).all())
    p3 = pre.reshape(3, 4, 96).clone().requires_grad_()
    t3 = log_thr.clone().requires_grad_()
    (B.jumprelu8(p3, t3, eps)[0] * w.reshape(3, 4, 96)).sum().backward()
    assert torch.equal(p3.grad.reshape(12, 96), p.grad) and torch.equal(t3.grad, t.grad)
    only = log_thr.clone().requires_grad_()
    B.jumprelu8(pre, only, eps)[1].sum().backward()       # the gate's gradient alone
    band = ((pre.double() - theta).abs() < eps).sum(0)
    torch.testing.assert_close(only.grad.double(), -band * theta / (2 * eps), rtol=1e-6, atol=0)
    e = torch.zeros(0, 96, device=DEV, requires_grad=True)
    te = log_thr.clone().requires_grad_()
    sum(o.sum() for o in B.jumprelu8(e, te, eps)).backward()
    assert e.grad.shape == (0, 96) and not te.grad.any()


def test_other_stream_and_captured_graph():
    """Calls on a side stream, and a captured save + weight gradient replayed on
    new values in the same buffers."""
    B = _pkg()
    x, g = torch.randn(130, 96, device=DEV), torch.randn(130, 264, device=DEV).bfloat16()
    want = B.checkpoint8(x).weight_grad(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = B.checkpoint8(x).weight_grad(g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):                                   # two graphs, no scratch in common
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = B.checkpoint8(x).weight_grad(g)
        graphs.append((gr, out))
    x.mul_(1.5).add_(0.25)
    want = B.checkpoint8(x).weight_grad(g)
    for gr, out in graphs:
        gr.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out, want)


def test_jumprelu8_captured_and_versions():
    """Forward and backward captured together and replayed on new values; results
    written into a caller's tensor count as in-place changes of it."""
    B = _pkg()
    pre = torch.randn(70, 640, device=DEV)
    lt = torch.full((640,), -0.5, device=DEV, requires_grad=True)
    gf = torch.randn(70, 640, device=DEV)

    def run():
        p = pre.detach().requires_grad_()
        feat, gate = B.jumprelu8(p, lt, 0.25)
        return (feat, gate, *torch.autograd.grad((feat, gate), (p, lt), (gf, gf)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = run()
    pre.mul_(0.7)
    gf.neg_()
    want = run()
    gr.replay()
    for a, b in zip(out, want):
        assert torch.equal(a, b)
    held = B.checkpoint8(pre)
    for out, write in ((torch.zeros(70, 640, device=DEV), lambda o: held.dequantize(out=o)),
                       (torch.zeros(640, 640, device=DEV), lambda o: held.weight_grad(gf, out=o))):
        w = torch.ones_like(out, requires_grad=True)
        loss = (w * out).sum()                    # saves out
        write(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_jumprelu8_is_differentiable_once():
    B = _pkg()
    pre = torch.randn(9, 40, device=DEV, requires_grad=True)
    lt = torch.zeros(40, device=DEV, requires_grad=True)
    plain = torch.autograd.grad(B.jumprelu8(pre, lt, 0.5)[0].sum(), (pre, lt))
    graphed = torch.autograd.grad(B.jumprelu8(pre, lt, 0.5)[0].sum(), (pre, lt), create_graph=True)
    for a, b in zip(plain, graphed):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):           # no graph of the gradients: nothing asks for one
        graphed[1].sum().backward()
    w = torch.ones(9, 40, device=DEV, requires_grad=True)
    graphed = torch.autograd.grad(B.jumprelu8(pre, lt, 0.5)[0], (pre, lt), w, create_graph=True)
    for a, b in zip(plain, graphed):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        graphed[1].sum().backward()


def test_offsets_past_32_bits():
    """45000 x 49152 elements, all but the last 40 rows zero (or off): those rows
    as a call on them alone gives them, in every output."""
    B = _pkg()
    T, F, n = 45000, 49152, 40
    gen = torch.Generator(device=DEV).manual_seed(7)
    tail = torch.randn(n, F, device=DEV, generator=gen).bfloat16()
    x = torch.zeros(T, F, device=DEV, dtype=torch.bfloat16)
    x[-n:] = tail
    held, small = B.checkpoint8(x), B.checkpoint8(tail)
    assert torch.equal(held.codes[-n:], small.codes) and torch.equal(held.steps[-n:], small.steps)
    assert torch.equal(held.dequantize()[-n:], small.dequantize())
    g = torch.randn(T, 24, device=DEV, generator=gen).bfloat16()
    got = held.weight_grad(g)
    v, gt = small.dequantize(torch.float32).double(), g[-n:].double()
    room = 2.0 ** -23 * (64 + T / 256) * (gt.abs().t() @ v.abs())
    assert bool(((got.double() - gt.t() @ v).abs() <= room).all())
    del held, got
    x.fill_(-9.0)
    x[-n:] = tail
    lt = torch.full((F,), -0.5, device=DEV, requires_grad=True)
    grad = torch.randn(n, F, device=DEV, generator=gen)
    gf = torch.ones(T, F, device=DEV)
    gf[-n:] = grad
    outs = []
    for p, gr in ((x, gf), (tail, grad)):
        p = p.requires_grad_()
        feat, gate = B.jumprelu8(p, lt, 0.25)
        outs.append((feat[-n:].clone(), gate[-n:].clone(),
                     *(t[-n:].clone() for t in torch.autograd.grad(
                         (feat, gate), (p, lt), (gr, torch.full((1, 1), 0.5, device=DEV).expand_as(gr))))))
        del feat, gate
    for a, b in zip(outs[0][:3], outs[1][:3]):
        assert torch.equal(a, b)
    # the same terms in other slabs: 2^-23 a term of theta / (2 eps) (|value grad| + 0.5)
    room = n * 2.0 ** -23 * 2 * (0.8 * 6 + 0.5)
    assert bool(((outs[0][3] - outs[1][3]).abs() <= room).all())


# ------------------------------------------------------------------ module
def _train_pass(sae, x, autocast):
    for p in sae.parameters():
        p.grad = None
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        pre = sae.encode_pre(x)
        pre.retain_grad()
        feat, gate = sae.jumprelu_with_gate(pre)
        x_hat = sae.decode(feat)
        loss = (x.float() - x_hat).square().mean() + 1e-3 * gate.sum(1).mean()
    loss.backward()
    return x_hat.detach(), feat.detach(), pre.grad.detach()


@pytest.mark.parametrize("autocast", [True, False])
@pytest.mark.parametrize("d,F,T", [(128, 512, 200), (96, 1000, 33), (256, 2048, 520)])
def test_module_with_8_bit_checkpoints(d, F, T, autocast):
    """The module's training pass with checkpoint_bits = 8: the same forward and
    the same gradients but for what the checkpoints round, which bounds the
    difference element by element (half a step of the saved value)."""
    B = _pkg()
    sae = B.make_sae(d, F, seed=1).cuda()
    with torch.no_grad():
        sae.log_threshold.fill_(np.log(0.6))
    sae.ste_bandwidth = 0.25
    x = 2 * torch.randn(T, d, device=DEV)
    ref = _train_pass(sae, x, autocast)
    g_ref = {n: p.grad.clone() for n, p in sae.named_parameters()}
    sae.checkpoint_bits = 8
    got = _train_pass(sae, x, autocast)
    g = {n: p.grad.clone() for n, p in sae.named_parameters()}
    for a, b in zip(ref, got):
        assert torch.equal(a, b)
    assert torch.equal(g["W_enc.bias"], g_ref["W_enc.bias"])
    assert torch.equal(g["b_dec"], g_ref["b_dec"])
    x_hat, feat, dpre = (t.double() for t in ref)

    def half_steps(v):
        a = B.checkpoint8(v)
        s = torch.exp2(a.steps.double() - 128).repeat_interleave(32, 1)
        return s[:, :v.shape[1]]

    xc = x - sae.b_dec.detach()
    xc = xc.bfloat16() if autocast else xc
    acts = feat.bfloat16() if autocast else feat.float()
    go = (2 / x.numel() * (x_hat - x.double())).abs()
    room = 2.0 ** -20                    # fp32 sums on either side, and go's own rounding
    lim = dpre.abs().t() @ half_steps(xc) + room * (dpre.abs().t() @ xc.double().abs())
    assert bool(((g["W_enc.weight"] - g_ref["W_enc.weight"]).double().abs() <= lim).all())
    lim = go.t() @ half_steps(acts) * (1 + 2.0 ** -7) + room * (go.t() @ acts.double().abs())
    assert bool(((g["W_dec.weight"] - g_ref["W_dec.weight"]).double().abs() <= lim).all())
    # threshold: the band's value is good to eps / 252, on grad_feat
    diff = (g["log_threshold"] - g_ref["log_threshold"]).double().abs()
    theta, eps = 0.6, 0.25
    W = (sae._shadow_dec if autocast else sae._dec_fm()).detach().double()
    gf = (go.bfloat16().double() if autocast else go) @ W.abs().t()
    assert bool((diff <= theta / (2 * eps) * (eps / 252) * gf.sum(0) * 1.02 + 1e-6).all())
    assert float(g["log_threshold"].abs().max()) > 0


def test_module_with_an_input_that_needs_a_gradient():
    """x's own gradient: its fp32 path keeps x, the rest is held in 8 bits."""
    B = _pkg()
    sae = B.make_sae(96, 512, seed=1).cuda()
    with torch.no_grad():
        sae.log_threshold.fill_(np.log(0.4))
    x = torch.randn(50, 96, device=DEV, requires_grad=True)
    grads = []
    for bits in (None, 8):
        sae.checkpoint_bits = bits
        x_hat, acts = sae(x)
        (x_hat.square().sum() + acts.sum()).backward()
        grads.append((x.grad.clone(), sae.W_enc.weight.grad.clone()))
        x.grad = None
        sae.zero_grad()
    assert torch.equal(grads[0][0], grads[1][0])        # gates and products are the same
    assert torch.equal(grads[0][1], grads[1][1])


def test_module_checkpoint_memory_and_refusals():
    B = _pkg()
    sae = B.make_sae(128, 8192, seed=0).cuda()
    x = torch.randn(1024, 128, device=DEV)

    def kept():
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        with torch.autocast("cuda", torch.bfloat16):
            x_hat, acts = sae(x)
        n = torch.cuda.memory_allocated() - base - acts.numel() * 4 - x_hat.numel() * 4
        return n

    kept()
    plain = kept()
    sae.checkpoint_bits = 8
    small = kept()
    elements = 1024 * 8192
    assert plain >= 4 * elements and small <= 2.3 * elements
    with pytest.raises(ValueError):
        sae.checkpoint_bits = 4
    with torch.autocast("cuda", torch.bfloat16):
        loss = sae(x)[0].sum()
    sae.ste_bandwidth = 0.3
    with pytest.raises(RuntimeError, match="ste_bandwidth"):
        loss.backward()
    with torch.no_grad():                       # nothing is kept, the plain path runs
        a = sae(x)
    for p in sae.parameters():                  # no parameter asks: nothing to keep
        p.requires_grad_(False)
    before = kept()
    sae.checkpoint_bits = None
    assert before <= kept()
    with torch.no_grad():
        b = sae(x)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("frozen", ["W_enc.weight", "W_dec.weight"])
def test_module_with_a_frozen_weight_keeps_nothing_for_it(frozen, bits):
    """The encoder's input and the decoder's are kept for their weight gradients alone:
    a frozen weight costs neither their bytes nor a product, and the other gradients
    are the same bits."""
    B = _pkg()
    sae = B.make_sae(1024, 8192, seed=0).cuda()
    sae.checkpoint_bits = bits
    T = 1024
    x = torch.randn(T, 1024, device=DEV)

    def run():
        for p in sae.parameters():
            p.grad = None
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        with torch.autocast("cuda", torch.bfloat16):
            x_hat, acts = sae(x)
        kept = torch.cuda.memory_allocated() - base - acts.numel() * 4 - x_hat.numel() * 4
        (x_hat.square().sum() + acts.sum()).backward()
        return kept, {n: p.grad for n, p in sae.named_parameters()}

    run()
    whole, want = run()
    dict(sae.named_parameters())[frozen].requires_grad_(False)
    less, got = run()
    assert got.pop(frozen) is None
    for n, g in got.items():
        assert torch.equal(g, want[n]), n
    elements = T * (1024 if frozen == "W_enc.weight" else 8192)
    assert whole - less >= elements * (1 if bits == 8 else 2)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("N", [1800, 1801])        # gradients read in place, or copied first
def test_weight_grad_of_codes_expanded_in_several_launches(N, transposed):
    """Many gradient columns of a wide checkpoint: the codes are expanded beforehand, a
    part of the tokens at a time, the last one shorter; later launches add to the first."""
    import ctypes
    B = _pkg()
    from sae_b200 import _lib as L
    T, D = 3700, 33000
    gen = torch.Generator(device=DEV).manual_seed(N)
    x = torch.randn(T, D, device=DEV, generator=gen).bfloat16()
    g = (torch.randn(T, N, device=DEV, generator=gen) * 1e-3).bfloat16()
    a = B.checkpoint8(x)
    need = ctypes.c_size_t(0)
    L.call("sae_b200_weight_grad8_workspace_bytes", T, D, g.data_ptr(), L.DTYPE_BF16, N, N,
           ctypes.byref(need))
    values = need.value - (0 if N % 8 == 0 else 2 * 1808 * (need.value // (2 * (1808 + 33024))))
    held = values // (2 * 33024)                     # tokens expanded at a time
    assert T / 4 < held < T / 2 and T % held != 0
    v, g64 = a.dequantize(torch.float32).double(), g.double()
    want = g64.t() @ v
    bound = 2.0 ** -23 * (64 + T / 256) * (g64.abs().t() @ v.abs())
    del v, g64
    base = torch.randn((D, N) if transposed else (N, D), device=DEV, generator=gen) * 1e-2
    got = a.weight_grad(g, transposed=transposed)
    acc = a.weight_grad(g, transposed=transposed, out=base.clone(), accumulate=True)
    turn = (lambda t: t.t()) if transposed else (lambda t: t)
    # each launch after the first rounds its sum with what is there
    room = bound + 2 * 2.0 ** -24 * (want.abs() + bound) + 1e-37
    assert bool(((turn(got).double() - want).abs() <= room).all())
    room = bound + 3 * 2.0 ** -24 * (want.abs() + bound + turn(base).double().abs()) + 1e-37
    assert bool(((turn(acc).double() - turn(base).double() - want).abs() <= room).all())
    assert torch.equal(a.weight_grad(g, transposed=transposed), got)


@pytest.mark.parametrize("base,unit", [(1.0, 2.0 ** -7), (1.0, 2.0 ** -15), (1.0, 2.0 ** -23),
                                       (1.0 + 2.0 ** -8, 2.0 ** -23)])
def test_weight_grad_uses_all_bits_of_fp32_gradients(base, unit):
    """Tokens in pairs whose gradients base + k unit and -base leave sum k unit v, over one
    stage of 64 tokens, in which the upper parts are added first, then the middle ones.

    Units of 2^-7 and 2^-15: products have 15 bits, and what the upper parts leave is at
    most 2^-8 sum |v| < 16, so every partial sum has 20 bits and is exact. base
    1 + 2^-8, k >= 0: the upper parts 1 and the middle ones 2^-8 cancel, the lower ones are
    k unit; exact. base 1, unit 2^-23: for k < 0 the upper part is 1 - 2^-8, so 2^-8 sum |v|
    is left until the lower parts are added, and each of their eight products of 16
    tokens may lose two units in the last place of that."""
    B = _pkg()
    gen = torch.Generator(device=DEV).manual_seed(2)
    v = torch.randint(-127, 128, (32, 160), device=DEV, generator=gen)
    v[:, ::32] = 127                                  # the step of every group is 1
    k = torch.randint(-100, 101, (32, 300), device=DEV, generator=gen)
    room = torch.zeros(160, device=DEV, dtype=torch.float64)
    if base != 1:
        k = k.abs()
    elif unit == 2.0 ** -23:
        room = 8 * 2 * 2.0 ** -23 * 2.0 ** -8 * v.abs().sum(0).double()
    x = v.repeat_interleave(2, 0).float()
    g = torch.empty(64, 300, device=DEV)
    g[0::2], g[1::2] = base + k * unit, -base
    assert torch.equal(g[0::2].double() - base, k * unit)       # held by fp32
    want = (k.t().double() @ v.double()) * unit
    for transposed in (False, True):
        got = B.checkpoint8(x).weight_grad(g, transposed=transposed)
        off = ((got.t() if transposed else got).double() - want).abs()
        assert bool((off <= room).all())


def test_no_wait_ran_out():
    """Kernels' waits are bounded; one that ran out, here or in a test before, is recorded."""
    B = _pkg()
    from sae_b200 import _lib as L
    x = torch.randn(500, 640, device=DEV)
    for g in (torch.randn(500, 700, device=DEV), torch.randn(500, 2000, device=DEV).bfloat16()):
        B.checkpoint8(x).weight_grad(g)
    assert L.device_status() == 0
