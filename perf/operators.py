"""Cases that measure the low-precision operators: sparse-autoencoder weights in 4 bits for
serving (encode4, reconstruct4) and activation checkpoints in 8 bits for training (checkpoint8,
weight_grad8, jumprelu8).

Each operator has a plain form in elementary torch operations (``own`` false), the calls a user
of the package makes (``own`` true), and its definition in 64 bits (``exact``).

Formats, shared by all three:

* 4-bit weights ``[F, d]``: a byte holds two columns, the even one in its low half, as q + 8 with q
  in [-7, 7]; ``group`` columns of a row share a bfloat16 scale with at most 5 significant bits.
* 8-bit checkpoints ``[T, D]``: 32 columns of a row share a step 2^k, the smallest (k >= -126) with
  max|x| 2^-k < 127.5; an element is held as rint(x 2^-k).
* JumpReLU checkpoints: with u = pre - theta, a byte holds ceil(126 u / eps) inside the band
  |u| < eps, 127 above it and -128 below it; inside the band it stands for the middle of its step.
"""
import math
import pathlib
import sys

import torch

own = False

GROUP8 = 32          # columns that share a step in an 8-bit checkpoint
BAND_STEPS = 126     # steps of a JumpReLU checkpoint in half a band


def _package():
    root = str(pathlib.Path(__file__).resolve().parents[1] / "event-aware-sae-trainer_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import sae_b200
    return sae_b200


# ------------------------------------------------------------------ cases
def listed():
    return [
        # Serving next to a decoding language model: one new token at the 1536 x 49152 dictionary.
        dict(name="reconstruct4_token", op="reconstruct4", T=1, d=1536, F=49152, group=64, l0=50,
             x="bf16"),
        # The smallest dictionary of the configurations, three float32 tokens: latency only.
        dict(name="reconstruct4_small", op="reconstruct4", T=3, d=256, F=8192, group=32, l0=50,
             x="f32"),
        # A batch of sequences, one token each, at the inference configuration's shape.
        dict(name="reconstruct4_batch", op="reconstruct4", T=128, d=2304, F=65536, group=64, l0=80,
             x="bf16"),
        # Feature monitoring of one token on the widest dictionary: a quarter gigabyte of weights.
        dict(name="encode4_token_wide", op="encode4", T=1, d=4096, F=131072, group=128, l0=64,
             x="bf16"),
        # A few sequences at once, an odd number of them.
        dict(name="encode4_batch", op="encode4", T=21, d=1536, F=49152, group=64, l0=50, x="bf16"),
        # A prompt of some hundred tokens.
        dict(name="encode4_prompt", op="encode4", T=300, d=1536, F=49152, group=64, l0=50,
             x="f32"),
        # One pool shard (32768 tokens), written in 8 bits and read back for a step.
        dict(name="checkpoint8_shard", op="checkpoint8", T=32768, d=1536, x="bf16"),
        # Ragged: columns that end inside a group, float32.
        dict(name="checkpoint8_ragged", op="checkpoint8", T=1000, d=777, x="f32"),
        # The encoder's weight gradient of a whole microbatch: the input saved in 8 bits.
        dict(name="weight_grad8_encoder", op="weight_grad8", T=32768, d=1536, N=49152,
             transposed=False, g="bf16", density=0.05),
        # The decoder's weight gradient of the small configuration: the activations saved in 8 bits
        # ([T, 8192]), float32 output gradients.
        dict(name="weight_grad8_decoder", op="weight_grad8", T=4096, d=8192, N=256,
             transposed=True, g="f32", density=1.0),
        # JumpReLU forward and backward; the gate's gradient is one number for all (sparsity loss).
        dict(name="jumprelu8_autocast", op="jumprelu8", T=4096, F=49152, pre="bf16", gate="scalar"),
        # A ragged float32 slab with a gradient for each gate.
        dict(name="jumprelu8_ragged", op="jumprelu8", T=517, F=9001, pre="f32", gate="full"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["reconstruct4", "encode4", "checkpoint8", "weight_grad8", "jumprelu8"])
    if op in ("reconstruct4", "encode4"):
        d = _log_int(rng, 128, 4096) // 2 * 2     # codes hold two columns to the byte
        F = _log_int(rng, 1000, 70000)
        T = _log_int(rng, 1, 512)
        return dict(op=op, T=T, d=d, F=F, group=rng.choice([32, 64, 128]),
                    l0=rng.randint(8, 120), x=rng.choice(["bf16", "f32"]))
    if op == "checkpoint8":
        return dict(op=op, T=_log_int(rng, 1, 32768), d=_log_int(rng, 31, 4096),
                    x=rng.choice(["bf16", "f32"]))
    if op == "weight_grad8":
        small, large = _log_int(rng, 100, 2304), _log_int(rng, 500, 33000)
        transposed = rng.random() < 0.5
        return dict(op=op, T=_log_int(rng, 16, 8192), d=large if transposed else small,
                    N=small if transposed else large, transposed=transposed,
                    g=rng.choice(["bf16", "bf16", "f32"]), density=rng.choice([0.02, 0.2, 1.0]))
    return dict(op=op, T=_log_int(rng, 1, 6000), F=_log_int(rng, 500, 33000),
                pre=rng.choice(["bf16", "f32"]), gate=rng.choice(["scalar", "full"]))


# ----------------------------------------------------------------- inputs
_DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _round_scale(s):
    """Up to the next number with 5 significant bits (a bfloat16)."""
    m, e = torch.frexp(s)
    return torch.ldexp(torch.ceil(m * 32) / 32, e).to(torch.bfloat16)


def _weights4(g, F, d, group):
    """Codes and scales of a random dictionary with unit rows."""
    w = torch.randn(F, d, generator=g, device="cuda")
    w /= w.norm(dim=1, keepdim=True)
    ng = -(-d // group)
    wp = torch.nn.functional.pad(w, (0, ng * group - d)).reshape(F, ng, group)
    scale = _round_scale(wp.abs().amax(2) / 7)
    q = torch.round(wp / scale.float().unsqueeze(2)).clamp(-7, 7).to(torch.int32) + 8
    q = q.reshape(F, ng * group)[:, :d]
    return (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8), scale


def _values4(codes, scale, group, dtype):
    """The weights that codes and scales stand for."""
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(codes.shape[0], -1).to(dtype) - 8
    return q * scale.to(dtype).repeat_interleave(group, 1)[:, :q.shape[1]]


def _tokens(g, T, d, b_dec, dtype):
    """Residual-stream rows: a LogNormal norm around a common bias."""
    x = torch.randn(T, d, generator=g, device="cuda")
    norm = torch.exp(math.log(60.0) + 0.4 * torch.randn(T, 1, generator=g, device="cuda"))
    return (x / x.norm(dim=1, keepdim=True) * norm + b_dec).to(dtype)


def _prepare_sae4(case, g):
    T, d, F, group = case["T"], case["d"], case["F"], case["group"]
    s = dict(case)
    s["enc"], s["enc_scale"] = _weights4(g, F, d, group)
    s["dec"], s["dec_scale"] = _weights4(g, F, d, group)
    s["b_enc"] = 0.1 * torch.randn(F, generator=g, device="cuda")
    s["b_dec"] = 0.5 * torch.randn(d, generator=g, device="cuda")
    s["tokens"] = _tokens(g, T, d, s["b_dec"], _DTYPE[case["x"]])
    # Thresholds that leave about l0 features of a token active, spread as trained ones are, and
    # clear of every pre-activation of these tokens: a value next to its threshold would pass or
    # fail by the order of a sum.
    pre = _pre64(s)
    base = pre.flatten().topk(min(pre.numel(), case["l0"] * T)).values[-1].clamp(min=1e-3)
    theta = base * torch.exp(0.1 * torch.randn(F, generator=g, device="cuda").double())
    best, best_gap = theta, torch.full_like(theta, -1.0)
    for k in range(8):
        cand = theta * (1 + 0.004 * k)
        gap = (pre - cand).abs().amin(0)
        best = torch.where(gap > best_gap, cand, best)
        best_gap = torch.maximum(gap, best_gap)
    s["log_threshold"] = best.log().float()
    if own:
        s["sae4"] = _package().B200SAE4.from_codes(
            s["enc"], s["enc_scale"], s["b_enc"], s["dec"], s["dec_scale"], s["b_dec"],
            s["log_threshold"], group=group)
    return s


def _prepare_checkpoint8(case, g):
    s = dict(case)
    bias = 0.5 * torch.randn(case["d"], generator=g, device="cuda")
    s["tokens"] = _tokens(g, case["T"], case["d"], bias, _DTYPE[case["x"]])
    return s


def _prepare_weight_grad8(case, g):
    s = dict(case)
    T, d, N = case["T"], case["d"], case["N"]
    x = torch.randn(T, d, generator=g, device="cuda")
    if case["transposed"]:     # activations: most are zero
        x = torch.relu(x - 1.5) * 3
    s["saved"] = x.to(torch.bfloat16)
    grad = torch.empty(T, N, device="cuda", dtype=_DTYPE[case["g"]])
    for t in range(0, T, 4096):
        n = min(4096, T - t)
        v = 1e-3 * torch.randn(n, N, generator=g, device="cuda")
        if case["density"] < 1:     # gated gradients: zero where the feature is off
            v *= torch.rand(n, N, generator=g, device="cuda") < case["density"]
        grad[t:t + n] = v.to(grad.dtype)
    s["grad"] = grad
    return s


def _prepare_jumprelu8(case, g):
    s = dict(case)
    T, F = case["T"], case["F"]
    s["eps"] = 0.125
    s["log_threshold"] = math.log(0.1) + 0.3 * torch.randn(F, generator=g, device="cuda")
    theta = s["log_threshold"].double().exp()
    pre = torch.empty(T, F, device="cuda", dtype=_DTYPE[case["pre"]])
    for t in range(0, T, 2048):
        n = min(2048, T - t)
        p = (0.3 * torch.randn(n, F, generator=g, device="cuda") - 0.5).to(pre.dtype)
        # An element on the border of a step would round by the last bit of a logarithm: off.
        at = (p.double() - theta) * (BAND_STEPS / s["eps"])
        p[((at - at.round()).abs() < 1e-3) & (at.abs() < BAND_STEPS + 1)] = -1.0
        pre[t:t + n] = p
    s["pre_act"] = pre.requires_grad_()
    s["log_threshold"].requires_grad_()
    s["grad_feat"] = 1e-3 * torch.randn(T, F, generator=g, device="cuda")
    gate = 1e-4 * torch.randn(1 if case["gate"] == "scalar" else T * F, generator=g, device="cuda")
    s["grad_gate"] = gate.expand(T, F) if case["gate"] == "scalar" else gate.reshape(T, F)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] in ("encode4", "reconstruct4"):
        return _prepare_sae4(case, g)
    return {"checkpoint8": _prepare_checkpoint8, "weight_grad8": _prepare_weight_grad8,
            "jumprelu8": _prepare_jumprelu8}[case["op"]](case, g)


# ------------------------------------------------------------ plain forms
def _plain_encode4(s):
    xc = (s["tokens"].float() - s["b_dec"]).to(torch.bfloat16).float()
    w = _values4(s["enc"], s["enc_scale"], s["group"], torch.float32)
    pre = xc @ w.t() + s["b_enc"]
    return torch.where(pre > s["log_threshold"].exp(), pre, torch.zeros_like(pre))


def _plain_reconstruct4(s):
    feat = _plain_encode4(s)
    w = _values4(s["dec"], s["dec_scale"], s["group"], torch.float32)
    return {"x_hat": feat @ w + s["b_dec"], "active": (feat > 0).sum(1, dtype=torch.int32)}


def _plain_values8(x):
    """The values that an 8-bit checkpoint of x holds, in float32."""
    T, d = x.shape
    ng = -(-d // GROUP8)
    v = torch.nn.functional.pad(x.float(), (0, ng * GROUP8 - d)).reshape(T, ng, GROUP8)
    m, e = torch.frexp(v.abs().amax(2, keepdim=True))
    k = torch.where(m < 127.5 / 128, e - 7, e - 6).clamp(min=-126)
    up = ((127 - k) << 23).to(torch.int32).view(torch.float32)       # 2^-k
    down = ((127 + k) << 23).to(torch.int32).view(torch.float32)     # 2^k
    return (torch.round(v * up) * down).reshape(T, ng * GROUP8)[:, :d]


def _plain_weight_grad8(s):
    v, g = _plain_values8(s["saved"]), s["grad"].float()
    return v.t() @ g if s["transposed"] else g.t() @ v


def _plain_jumprelu8(s):
    pre, eps = s["pre_act"].detach().float(), s["eps"]
    theta = s["log_threshold"].detach().exp()
    u = pre - theta
    gate, band = pre > theta, u.abs() < eps
    zero = torch.zeros((), device=pre.device)
    code = torch.ceil(u * (BAND_STEPS / eps))
    code = torch.where(gate, code.clamp(1, BAND_STEPS), code.clamp(1 - BAND_STEPS, 0))
    held = theta + (code - 0.5) * (eps / BAND_STEPS)
    gf, gg = s["grad_feat"], s["grad_gate"]
    ste = torch.where(band, held * gf + gg, zero).sum(0, dtype=torch.float64)
    return {"feat": torch.where(gate, pre, zero), "gate": gate.float(),
            "grad_pre": torch.where(gate, gf, zero).to(s["pre_act"].dtype),
            "grad_log_threshold": (-ste / (2 * eps) * theta.double()).float()}


def _run_own(s):
    B = _package()
    op = s["op"]
    if op == "reconstruct4":
        x_hat, active = s["sae4"].reconstruct(s["tokens"])
        return {"x_hat": x_hat, "active": active}
    if op == "encode4":
        return s["sae4"].encode(s["tokens"])
    if op == "checkpoint8":
        return B.checkpoint8(s["tokens"]).dequantize(torch.bfloat16)
    if op == "weight_grad8":
        return B.checkpoint8(s["saved"]).weight_grad(s["grad"], transposed=s["transposed"])
    feat, gate = B.jumprelu8(s["pre_act"], s["log_threshold"], s["eps"])
    gp, gt = torch.autograd.grad((feat, gate), (s["pre_act"], s["log_threshold"]),
                                 (s["grad_feat"], s["grad_gate"]))
    return {"feat": feat, "gate": gate, "grad_pre": gp, "grad_log_threshold": gt}


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "checkpoint8":
        return _plain_values8(state["tokens"]).to(torch.bfloat16)
    return {"reconstruct4": _plain_reconstruct4, "encode4": _plain_encode4,
            "weight_grad8": _plain_weight_grad8, "jumprelu8": _plain_jumprelu8}[op](state)


# ------------------------------------------------------------ definitions
def _pre64(s):
    xc = (s["tokens"].float() - s["b_dec"]).to(torch.bfloat16).double()
    w = _values4(s["enc"], s["enc_scale"], s["group"], torch.float64)
    return xc @ w.t() + s["b_enc"].double()


def _exact_values8(x):
    T, d = x.shape
    ng = -(-d // GROUP8)
    v = torch.nn.functional.pad(x.double(), (0, ng * GROUP8 - d)).reshape(T, ng, GROUP8)
    big = v.abs().amax(2, keepdim=True).clamp(min=2.0 ** -140)
    k = torch.floor(torch.log2(big)) - 6
    for _ in range(2):     # log2 may be off by one next to a power of two
        k = torch.where(big * torch.exp2(-k) >= 127.5, k + 1, k)
        k = torch.where(big * torch.exp2(1 - k) < 127.5, k - 1, k)
    k = k.clamp(min=-126)
    return (torch.round(v * torch.exp2(-k)) * torch.exp2(k)).reshape(T, ng * GROUP8)[:, :d]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("encode4", "reconstruct4"):
        pre = _pre64(s)
        feat = pre * (pre > s["log_threshold"].double().exp())
        if s["op"] == "encode4":
            return feat
        w = _values4(s["dec"], s["dec_scale"], s["group"], torch.float64)
        return {"x_hat": feat @ w + s["b_dec"].double(),
                "active": (feat != 0).sum(1, dtype=torch.int32)}
    if s["op"] == "checkpoint8":
        return _exact_values8(s["tokens"])
    if s["op"] == "weight_grad8":
        v, g = _exact_values8(s["saved"]), s["grad"].double()
        return v.t() @ g if s["transposed"] else g.t() @ v
    eps, theta = s["eps"], s["log_threshold"].detach().double().exp()
    pre = s["pre_act"].detach()
    out = {"feat": pre.float(), "gate": None, "grad_pre": s["grad_feat"].clone(),
           "grad_log_threshold": torch.zeros_like(theta)}
    for t in range(0, pre.shape[0], 2048):
        r = slice(t, t + 2048)
        u = pre[r].double() - theta
        out["feat"][r] *= u > 0
        out["grad_pre"][r] *= u > 0
        held = theta + (torch.ceil(u * BAND_STEPS / eps) - 0.5) * eps / BAND_STEPS
        ste = held * s["grad_feat"][r].double() + s["grad_gate"][r].double()
        out["grad_log_threshold"] -= (ste * (u.abs() < eps)).sum(0) * theta / (2 * eps)
    out["gate"] = (out["feat"] != 0).float()
    return out


# ------------------------------------------------------------------- work
def work(case):
    T = case["T"]
    size = {"bf16": 2, "f32": 4}
    if case["op"] in ("encode4", "reconstruct4"):
        d, F, group = case["d"], case["F"], case["group"]
        row = d / 2 + 2 * math.ceil(d / group)
        n = F * row + 8 * F + 4 * d + T * d * size[case["x"]]
        flops = 2.0 * T * F * d
        if case["op"] == "encode4":
            return {"bytes": n + 4.0 * T * F, "flops": flops}
        rows = F * (1 - (1 - case["l0"] / F) ** T)      # decoder rows that some token needs
        return {"bytes": n + rows * row + 4.0 * T * (d + 1),
                "flops": flops + 2.0 * T * case["l0"] * d}
    if case["op"] == "checkpoint8":
        return {"bytes": T * case["d"] * (size[case["x"]] + 2.0), "flops": 0.0}
    if case["op"] == "weight_grad8":
        d, N = case["d"], case["N"]
        return {"bytes": T * d * 2.0 + T * N * size[case["g"]] + 4.0 * d * N,
                "flops": 2.0 * T * d * N}
    F, n = case["F"], size[case["pre"]]
    # pre read and its gradient written, feat and gate written, grad_feat (and each gate's) read
    return {"bytes": T * F * (2.0 * n + 12 + (4 if case["gate"] == "full" else 0)) + 16.0 * F,
            "flops": 0.0}
