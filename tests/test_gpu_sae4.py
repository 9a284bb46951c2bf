"""Serving from 4-bit weights against the definition in 64 bits.

Codes are whole numbers and have to be equal. The products q s xc are exact in
fp32, so a pre-activation may be off by 2^-23 (64 + d / 256) sum_k |w xc| -- the
16-column products of a 256-column stretch may each lose two units in the last
place of the running sum, and the stretches are added in fp32 -- plus its
rounding with b_enc. The decoder's sums are plain fp32: 2^-24 (L0 + 4)
sum |feat w|, on top of what the features are off by.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _pkg():
    import sae_b200
    return sae_b200


def unpack(codes, scales, group):
    c = codes.cpu().numpy()
    q = np.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1).astype(np.float64) - 8
    s = scales.float().cpu().numpy().astype(np.float64)
    return q * np.repeat(s, group, 1)[:, :q.shape[1]]


class Case:
    def __init__(self, d, F, group, seed=0, theta=0.8):
        B = _pkg()
        g = torch.Generator(device=DEV).manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
        self.d, self.F, self.group = d, F, group
        enc, dec = rn(F, d) / d ** 0.5, rn(F, d) / d ** 0.5
        self.enc_c, self.dec_c = B.quantize4_rows(enc, group), B.quantize4_rows(dec, group)
        self.b_enc, self.b_dec = 0.1 * rn(F), 0.5 * rn(d)
        self.log_thr = np.log(theta) + 0.2 * rn(F)
        self.sae = B.B200SAE4.from_codes(*self.enc_c, self.b_enc, *self.dec_c, self.b_dec,
                                         self.log_thr, group=group)
        self.W, self.D = unpack(*self.enc_c, group), unpack(*self.dec_c, group)
        self.gen = g

    def tokens(self, T, dtype):
        return (torch.randn(T, self.d, device=DEV, generator=self.gen) + self.b_dec).to(dtype)

    def pre(self, x):
        xc = (x.float() - self.b_dec).bfloat16().double().cpu().numpy()
        b = self.b_enc.double().cpu().numpy()
        pre = xc @ self.W.T + b
        room = 2.0 ** -23 * (64 + self.d / 256) * (np.abs(xc) @ np.abs(self.W).T) \
            + 2.0 ** -23 * (np.abs(b) + np.abs(pre)) + 1e-37
        return pre, room

    def theta(self):
        return self.log_thr.exp().double().cpu().numpy()

    def decoded(self, feat, feat_room):
        x = feat @ self.D + self.b_dec.double().cpu().numpy()
        n = (feat != 0).sum(1, keepdims=True)
        size = np.abs(feat) @ np.abs(self.D)
        return x, 2.0 ** -24 * (n + 4) * size + feat_room @ np.abs(self.D) + 2.0 ** -23 * np.abs(x) + 1e-37


def np64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("F,d", [(1, 2), (3, 30), (16, 64), (33, 130), (40, 300)])
def test_quantize_rows(F, d, group):
    B = _pkg()
    g = torch.Generator(device=DEV).manual_seed(F + d)
    W = torch.randn(F, d, device=DEV, generator=g) * torch.exp(
        3 * torch.randn(F, 1, device=DEV, generator=g))
    W[0, : d // 2] = 0
    codes, scales = B.quantize4_rows(W, group)
    w = W.cpu().numpy()
    for f in range(F):
        for k in range(scales.shape[1]):
            part = w[f, k * group:(k + 1) * group]
            s = float(scales[f, k])
            amax = np.float32(np.abs(part).max())
            m, e = np.frexp(np.float32(amax / np.float32(7)))
            want = max(np.ldexp(np.ceil(np.float64(m) * 32) / 32, int(e)), 2.0 ** -100)
            assert s == want
            q = np.clip(np.rint(part / np.float32(s)), -7, 7)
            got = unpack(codes[f:f + 1], scales[f:f + 1], group)[0, k * group:(k + 1) * group]
            np.testing.assert_array_equal(got, q.astype(np.float64) * s)
            assert np.abs(got - part).max() <= s * (0.5 + 2.0 ** -22)


SHAPES = [(64, 16, 64), (2, 1, 32), (30, 17, 32), (66, 33, 32), (130, 250, 64), (300, 1000, 128),
          (768, 513, 64), (1536, 2048, 64), (322, 4800, 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 33, 64, 128, 129, 300])
@pytest.mark.parametrize("d,F,group", SHAPES)
def test_encode(d, F, group, T, dtype):
    c = Case(d, F, group, seed=d + F)
    x = c.tokens(T, dtype)
    pre, room = c.pre(x)
    got = np64(c.sae.encode_pre(x))
    assert (np.abs(got - pre) <= room).all()
    th = c.theta()
    feat = np64(c.sae.encode(x))
    clear = np.abs(pre - th) > room + 2.0 ** -22 * th
    np.testing.assert_array_equal((feat != 0)[clear], (pre > th)[clear])
    assert (np.abs(feat - np.where(feat != 0, pre, 0)) <= room).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 5, 24, 70])
@pytest.mark.parametrize("d,F,group", SHAPES)
def test_reconstruct_is_encode_then_decode(d, F, group, T, dtype):
    """The run of them together: reconstruct, and the features edited between
    encode and decode as for steering."""
    c = Case(d, F, group, seed=3)
    x = c.tokens(T, dtype)
    feat = c.sae.encode(x)
    fired = torch.zeros(F, device=DEV, dtype=torch.uint8)
    fired[-1] = 1
    x_hat, counts = c.sae.reconstruct(x, fired)
    assert counts.dtype == torch.int32 and x_hat.dtype == torch.float32
    assert torch.equal(counts, (feat != 0).sum(1, dtype=torch.int32))
    want_fired = (feat != 0).any(0).to(torch.uint8)
    want_fired[-1] = 1
    assert torch.equal(fired, want_fired)
    want, room = c.decoded(np64(feat), np.zeros(feat.shape))
    assert (np.abs(np64(x_hat) - want) <= room).all()
    assert torch.equal(c.sae.decode(feat), x_hat)          # the same rows in the same order
    assert torch.equal(c.sae.reconstruct(x)[0], x_hat)
    steered = feat.clone()
    steered[:, F // 2] = 4.0
    want, room = c.decoded(np64(steered), np.zeros(feat.shape))
    assert (np.abs(np64(c.sae.decode(steered)) - want) <= room).all()


@pytest.mark.parametrize("d,F", [(96, 5000), (520, 3001)])
def test_decode_empty_dense_and_non_finite_rows(d, F):
    c = Case(d, F, 32)
    acts = torch.randn(6, F, device=DEV)
    acts[0] = 0                                  # nothing active: b_dec alone
    acts[1, 1:] = 0
    acts[2, :-1] = 0
    got = c.sae.decode(acts)
    assert torch.equal(got[0], c.b_dec)
    want, room = c.decoded(np64(acts), np.zeros(acts.shape))
    assert (np.abs(np64(got) - want) <= room).all()    # rows 3..5 have all features active
    acts[3, 7] = float("nan")
    again = c.sae.decode(acts)
    assert bool(again[3].isnan().all()) and torch.equal(again[4:], got[4:])
    wide = torch.zeros(6, F + 11, device=DEV)
    wide[:, 3:3 + F] = acts
    assert torch.equal(c.sae.decode(wide[:, 3:3 + F])[4:], got[4:])


def test_thresholds_that_close_or_open_every_gate():
    c = Case(128, 300, 64)
    x = c.tokens(5, torch.float32)
    from sae_b200 import B200SAE4
    shut = B200SAE4.from_codes(*c.enc_c, c.b_enc, *c.dec_c, c.b_dec,
                               torch.full((300,), float("inf"), device=DEV), group=64)
    x_hat, counts = shut.reconstruct(x)
    assert not counts.any() and torch.equal(x_hat, c.b_dec.expand(5, 128))
    assert not shut.encode(x).any()
    wide = B200SAE4.from_codes(*c.enc_c, c.b_enc, *c.dec_c, c.b_dec,
                               torch.full((300,), float("-inf"), device=DEV), group=64)
    assert torch.equal(wide.encode(x), torch.relu(wide.encode_pre(x)))
    x[2, 5] = float("nan")                       # one token's NaN stays with it
    a, b = c.sae.reconstruct(x), c.sae.reconstruct(torch.where(x.isnan(), 0.0, x))
    assert bool(a[0][2].isnan().all())
    keep = [0, 1, 3, 4]
    assert torch.equal(a[0][keep], b[0][keep]) and torch.equal(a[1][keep], b[1][keep])


def test_no_tokens_strides_and_many_tokens():
    c = Case(128, 640, 64)
    for T in (0,):
        x_hat, counts = c.sae.reconstruct(torch.empty(T, 128, device=DEV))
        assert x_hat.shape == (0, 128) and counts.shape == (0,)
        assert c.sae.encode(torch.empty(T, 128, device=DEV)).shape == (0, 640)
        assert c.sae.decode(torch.empty(T, 640, device=DEV)).shape == (0, 128)
    big = c.tokens(2500, torch.bfloat16)
    x_hat, counts = c.sae.reconstruct(big)
    feat = c.sae.encode(big)
    assert torch.equal(counts, (feat != 0).sum(1, dtype=torch.int32))
    assert torch.equal(c.sae.decode(feat), x_hat)
    wide = torch.zeros(40, 300, device=DEV, dtype=torch.bfloat16)
    wide[:, 5:133] = big[:40]
    assert torch.equal(c.sae.encode(wide[:, 5:133]), c.sae.encode(big[:40].contiguous()))
    assert torch.equal(c.sae.encode(wide[::3, 5:133]), c.sae.encode(big[:40:3].contiguous()))
    assert torch.equal(c.sae.encode(big[:40].t().contiguous().t()), c.sae.encode(big[:40].contiguous()))


def test_quantize4_of_a_module_matches_its_own_reconstruction():
    """quantize4(sae): the 4-bit copy's x_hat is off from the module's by what
    the weights were rounded by -- half a scale each."""
    B = _pkg()
    sae = B.make_sae(256, 2048, seed=2).cuda()
    with torch.no_grad():
        sae.log_threshold.fill_(np.log(0.5))
        sae.b_dec.normal_()
    for group in (32, 64, 128):
        q = B.quantize4(sae, group)
        assert q.nbytes < 0.36 * 2 * 2048 * 256 * 2
        x = torch.randn(50, 256, device=DEV) + sae.b_dec.detach()
        codes, scales = B.quantize4_rows(sae.W_enc.weight, group)
        half = np.repeat(np64(scales), group, 1)[:, :256] * 0.51
        xc = np64((x - sae.b_dec).bfloat16())
        room = np.abs(xc) @ half.T + 1e-4
        with torch.no_grad():
            plain = xc @ np64(sae.W_enc.weight).T + np64(sae.W_enc.bias)
        assert (np.abs(np64(q.encode_pre(x)) - plain) <= room).all()
    with pytest.raises(ValueError):
        B.quantize4(sae, 48)
    with torch.no_grad():
        sae.W_enc.weight[3, 4] = float("nan")
    with pytest.raises(ValueError, match="finite"):
        B.quantize4(sae)


def test_from_codes_refusals():
    B = _pkg()
    c = Case(64, 48, 64)
    args = lambda: [*c.enc_c, c.b_enc, *c.dec_c, c.b_dec, c.log_thr]  # noqa: E731
    def but(i, t, **kw):
        a = args()
        a[i] = t
        with pytest.raises((ValueError, RuntimeError)):
            B.B200SAE4.from_codes(*a, **kw)
    but(0, c.enc_c[0][:, :-1])
    but(0, c.enc_c[0].to(torch.int8))
    but(1, c.enc_c[1].float())
    but(1, torch.full_like(c.enc_c[1], 1 + 2.0 ** -7))      # 8 significant bits
    but(1, torch.full_like(c.enc_c[1], float("nan")))
    but(1, -c.enc_c[1])
    but(1, torch.full_like(c.enc_c[1], 2.0 ** 61))
    but(2, c.b_enc[:-1])
    but(6, c.log_thr[:-1])
    but(6, torch.full_like(c.log_thr, float("nan")))
    but(5, c.b_dec.cpu())
    x = c.tokens(2, torch.float32)
    for bad in (x[:, :-1], x.reshape(1, 2, 64), x.half(), x.cpu()):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            c.sae.reconstruct(bad)
    with pytest.raises(ValueError):
        c.sae.reconstruct(x, torch.zeros(48, device=DEV))


def test_two_streams_and_captured_graphs():
    """Two streams at once on one handle, and two captured graphs replayed on
    new tokens: no scratch in common, the same bits as the plain calls."""
    c = Case(512, 4096, 64)
    xa, xb = c.tokens(3, torch.bfloat16), c.tokens(40, torch.bfloat16)
    wa, wb = c.sae.reconstruct(xa)[0], c.sae.reconstruct(xb)[0]
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (sa, sb):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        with torch.cuda.stream(sa):
            ga = c.sae.reconstruct(xa)[0]
        with torch.cuda.stream(sb):
            gb = c.sae.reconstruct(xb)[0]
        torch.cuda.synchronize()
        assert torch.equal(ga, wa) and torch.equal(gb, wb)
    graphs = []
    for x in (xa, xb):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c.sae.reconstruct(x)
        graphs.append((g, out))
    xa.copy_(c.tokens(3, torch.bfloat16))
    xb.copy_(c.tokens(40, torch.bfloat16))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for x, (_, out) in zip((xa, xb), graphs):
        want = c.sae.reconstruct(x)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("T", [1, 4, 6])
def test_an_outlier_costs_other_columns_no_precision(T):
    """A token whose largest element meets only zero weights: what is left is good
    to 2^-31 of that element in the few-token kernel's fixed point, and to the
    bounds above besides."""
    from sae_b200 import B200SAE4
    c = Case(256, 700, 64)
    codes = c.enc_c[0].clone()
    codes[:, 5] = (codes[:, 5] & 0xf0) | 8           # column 10: q = 0
    sae = B200SAE4.from_codes(codes, c.enc_c[1], c.b_enc, *c.dec_c, c.b_dec, c.log_thr, group=64)
    c.W = unpack(codes, c.enc_c[1], 64)
    x = c.tokens(T, torch.float32)
    pre, room = c.pre(x)
    x[:, 10] = 30000.0
    fixed = 2.0 ** -31 * 2 * 30000 * np.abs(c.W).sum(1)
    assert (np.abs(np64(sae.encode_pre(x)) - pre) <= room + fixed).all()


@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("d,F,group", [(12288, 100, 64), (12288, 40, 32), (8000, 1000, 128)])
def test_widest_inputs(d, F, group, T):
    c = Case(d, F, group)
    x = c.tokens(T, torch.bfloat16)
    pre, room = c.pre(x)
    assert (np.abs(np64(c.sae.encode_pre(x)) - pre) <= room).all()
    feat = c.sae.encode(x)
    want, lim = c.decoded(np64(feat), np.zeros(feat.shape))
    assert (np.abs(np64(c.sae.reconstruct(x)[0]) - want) <= lim).all()


def test_a_token_is_summed_the_same_in_any_batch():
    """decode: a token's result depends on its own active features alone, few or
    thousands, alone or in a batch."""
    c = Case(1100, 9000, 64)
    acts = torch.zeros(300, 9000, device=DEV)
    for t, n in enumerate([0, 1, 5, 190, 191, 192, 193, 194, 1000, 1025, 4000, 9000]):
        at = torch.randperm(9000, device=DEV, generator=c.gen)[:n]
        acts[t * 20, at] = torch.randn(n, device=DEV, generator=c.gen)
    whole = c.sae.decode(acts)
    want, room = c.decoded(np64(acts), np.zeros(acts.shape))
    assert (np.abs(np64(whole) - want) <= room).all()
    for t in range(0, 240, 20):
        assert torch.equal(c.sae.decode(acts[t:t + 1])[0], whole[t])


def test_offsets_past_32_bits():
    """45000 x 49152 features: the last tokens' as a call on them alone gives them."""
    c = Case(64, 49152, 64, theta=4.0)
    x = c.tokens(45000, torch.bfloat16)
    feat = c.sae.encode(x)
    tail = x[-40:].contiguous()
    pre, room = c.pre(tail)
    got, theta = np64(feat[-40:]), c.theta()
    clear = np.abs(pre - theta) > room + 2.0 ** -22 * theta
    want = np.where(pre > theta, pre, 0.0)
    assert (np.abs(got - want) <= room)[clear].all() and clear.mean() > 0.999
    x_hat = c.sae.decode(feat)
    assert torch.equal(x_hat[-40:], c.sae.decode(feat[-40:].contiguous()))


def test_a_new_handle_is_ready_for_any_stream():
    B = _pkg()
    c = Case(1024, 30000, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sae = B.B200SAE4.from_codes(*c.enc_c, c.b_enc, *c.dec_c, c.b_dec, c.log_thr, group=64)
    assert s.query()
    x = c.tokens(7, torch.float32)
    assert torch.equal(sae.encode_pre(x), c.sae.encode_pre(x))


@pytest.mark.parametrize("d,F,group,T", [(1536, 49152, 64, 300), (256, 70000, 32, 256),
                                         (1536, 49152, 32, 3), (1536, 49152, 64, 21)])
def test_more_feature_tiles_than_sms(d, F, group, T):
    """An SM goes on to further tiles while the last one's features are being stored:
    every call gives the same bits, within the bound."""
    B = _pkg()
    gen = torch.Generator(device=DEV).manual_seed(d + F + T)
    codes, scales = B.quantize4_rows(torch.randn(F, d, device=DEV, generator=gen) / d ** 0.5, group)
    sae = B.B200SAE4.from_codes(codes, scales, torch.zeros(F, device=DEV), codes, scales,
                                torch.zeros(d, device=DEV), torch.zeros(F, device=DEV), group=group)
    x = torch.randn(T, d, device=DEV, generator=gen).bfloat16()
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(F, d).double() - 8
    w = q * scales.double().repeat_interleave(group, 1)[:, :d]
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    del q, w
    room = 2.0 ** -23 * (64 + d / 256) * size + 2.0 ** -23 * want.abs() + 1e-37
    other = torch.empty(256 << 20, device=DEV, dtype=torch.uint8)
    first = sae.encode_pre(x)
    assert bool(((first.double() - want).abs() <= room).all())
    for _ in range(5):
        other.zero_()                    # the weights leave the L2 cache
        assert torch.equal(sae.encode_pre(x), first)


@pytest.mark.parametrize("T", [3, 4, 1027])
@pytest.mark.parametrize("d,F,group", [(9300, 6000, 32), (10000, 28000, 64), (10176, 25000, 128)])
def test_wide_inputs_of_three_and_four_tokens(d, F, group, T):
    """Widths at which four tokens, all of an SM's warps and their buffers do not fit
    together: fewer warps share a tile then. reconstruct of 1027 tokens ends with three."""
    B = _pkg()
    gen = torch.Generator(device=DEV).manual_seed(d + F)
    rows = lambda: B.quantize4_rows(torch.randn(F, d, device=DEV, generator=gen) / d ** 0.5, group)  # noqa: E731
    enc, dec = rows(), rows()
    b_enc = torch.randn(F, device=DEV, generator=gen)
    b_dec = torch.randn(d, device=DEV, generator=gen)
    sae = B.B200SAE4.from_codes(*enc, b_enc, *dec, b_dec, torch.full((F,), np.log(3.0), device=DEV),
                                group=group)
    x = torch.randn(T, d, device=DEV, generator=gen).bfloat16()
    x_hat, counts = sae.reconstruct(x)
    x, x_hat, counts = x[-3:], x_hat[-3:], counts[-3:]
    pre, feat = sae.encode_pre(x), sae.encode(x)
    assert torch.equal(feat, torch.where(pre > sae._theta, pre, 0.0))

    def weights(codes, scales):
        q = torch.stack((codes & 15, codes >> 4), 2).reshape(F, d).double() - 8
        return q * scales.double().repeat_interleave(group, 1)[:, :d]

    xc = (x.float() - b_dec).bfloat16().double()
    w = weights(*enc)
    want = xc @ w.t() + b_enc.double()
    room = 2.0 ** -23 * (64 + d / 256) * (xc.abs() @ w.abs().t()) + 2.0 ** -23 * (
        b_enc.double().abs() + want.abs()) + 1e-37
    assert bool(((pre.double() - want).abs() <= room).all())
    assert torch.equal(counts, (feat != 0).sum(1, dtype=torch.int32))
    w = weights(*dec)
    want = feat.double() @ w + b_dec.double()
    room = 2.0 ** -24 * (counts[:, None] + 4) * (feat.double().abs() @ w.abs()) \
        + 2.0 ** -23 * want.abs() + 1e-37
    assert bool(((x_hat.double() - want).abs() <= room).all())


def test_no_wait_ran_out():
    """Kernels' waits are bounded; one that ran out, here or in a test before, is recorded."""
    from sae_b200 import _lib as L
    c = Case(512, 4096, 64)
    for T in (1, 4, 40):
        c.sae.reconstruct(c.tokens(T, torch.bfloat16))
    assert L.device_status() == 0
