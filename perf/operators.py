"""Operators around the attention of a video transformer's layer, as cases that can be timed and compared.

  window    attention of a query chunk with a sliding window and first tokens that stay visible (ops.flash_window)
  rope      per-head norm of queries and keys and rotary positions on three axes (ops.norm_rope_grid, and its gradients)
  quantize  the rows of an attention state written in 8 bits, and read back (ops.quantize_rows, ops.dequantize_rows)
  merge     cached states in 8 bits merged with fresh ones, into a result or into a block of the cache (ops.merge_states)

With `own` false, `run` computes them by elementary torch operations in 32 bits (angles in 64); with `own` true it calls
the package.
"""
import math

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}        # largest magnitude of a code
SMALLEST_EXPONENT = 8


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # One token of a stream against its rolling cache: a window of 4096 positions and 256 first tokens.  Latency counts.
        dict(name="window_token", kind="window", B=1, Sq=1, Sk=8193, H=24, Hk=24, D=128, left=4095, right=0, sinks=256, ragged=False),
        # Three new tokens each of seven streams, caches of different lengths, four query heads to a key head.
        dict(name="window_tokens_ragged", kind="window", B=7, Sq=3, Sk=5003, H=32, Hk=8, D=64, left=2999, right=0, sinks=13, ragged=True),
        # The next latent frame (30 x 45 tokens) of a stream against the 4 frames before it and the 226 text tokens.
        dict(name="window_frame", kind="window", B=2, Sq=1350, Sk=17776, H=48, Hk=48, D=64, left=6749, right=1349, sinks=226, ragged=False),
        # The whole CogVideoX sequence (226 text + 13 x 1350 tokens), each token seeing a latent frame either way and the text.
        dict(name="window_cogvideox", kind="window", B=2, Sq=17776, Sk=17776, H=48, Hk=48, D=64, left=1350, right=1350, sinks=226, ragged=False),
        # A quarter of HunyuanVideo's 720p sequence with windows of a latent frame (45 x 80 tokens) either way.  The largest.
        dict(name="window_hunyuan", kind="window", B=1, Sq=29764, Sk=29764, H=24, Hk=24, D=128, left=3600, right=3600, sinks=256, ragged=False),
        # A toy layer in fp32, gradients: launches are all there is.
        dict(name="rope_small_grad", kind="rope", grad=True, B=1, H=4, D=64, text=7, T=3, Y=5, X=9, pad=2, dt=16, dy=24, rms=False, type="f32"),
        # CogVideoX: layer norm of each head, 13 x 30 x 45 latent positions behind 226 text tokens.
        dict(name="rope_cogvideox", kind="rope", grad=False, B=2, H=48, D=64, text=226, T=13, Y=30, X=45, pad=0, dt=16, dy=24, rms=False, type="bf16"),
        # HunyuanVideo's heads under RMS norm, nine latent frames of 45 x 80 on one rank: the gradients of a training step.
        dict(name="rope_hunyuan_grad", kind="rope", grad=True, B=1, H=24, D=128, text=256, T=9, Y=45, X=80, pad=25, dt=16, dy=56, rms=True, type="bf16"),
        # A CogVideoX chunk's state goes to the cache in int8 and is read back.
        dict(name="quantize_cogvideox", kind="quantize", B=2, S=2222, H=48, D=64, type="bf16", code="int8"),
        # The cache write of a HunyuanVideo chunk in fp32, as e4m3.
        dict(name="quantize_hunyuan", kind="quantize", B=1, S=14882, H=24, D=128, type="f32", code="e4m3"),
        # HunyuanVideo on one rank of 8: its own fresh state and seven blocks of an e4m3 cache give the layer's bf16 result.
        dict(name="merge_hunyuan", kind="merge", B=1, S=14882, H=24, D=128, cached=7, fresh=1, code="e4m3", to="bf16"),
        # CogVideoX, the cache taken to a coarser stride: four int8 blocks become one.
        dict(name="merge_blocks_cogvideox", kind="merge", B=2, S=2222, H=48, D=64, cached=4, fresh=0, code="int8", to="code"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_window(rng):
    D = rng.choice((64, 128))
    Hk, group = rng.choice(((1, 8), (4, 1), (8, 4), (12, 2), (24, 1), (48, 1)))
    B = rng.choice((1, 1, 2, 3))
    Sk = _log_int(rng, 300, 30000)
    Sq = rng.choice((1, _log_int(rng, 1, 16), _log_int(rng, 16, Sk), Sk))
    left = _log_int(rng, 32, 4000)
    right = rng.choice((0, left, _log_int(rng, 32, 4000)))
    case = dict(kind="window", B=B, Sq=min(Sq, Sk), Sk=Sk, H=Hk * group, Hk=Hk, D=D, left=left, right=right,
                sinks=rng.choice((0, rng.randrange(1, 64), rng.randrange(64, 300))), ragged=B > 1 and rng.random() < 0.5)
    most = work(listed()[4])["flops"]
    while work(case)["flops"] > most or case["B"] * case["Hk"] * case["Sk"] * case["D"] > 29764 * 24 * 128 * 4:
        case["Sk"] = case["Sk"] * 3 // 4
        case["Sq"] = min(case["Sq"], case["Sk"])
    return case


def _draw_rope(rng):
    D = rng.choice((64, 128))
    case = dict(kind="rope", grad=rng.random() < 0.5, B=rng.choice((1, 2)), H=rng.choice((1, 3, 8, 24, 48)), D=D,
                text=rng.choice((0, rng.randrange(1, 300))), T=rng.randrange(1, 14), Y=_log_int(rng, 2, 45), X=_log_int(rng, 3, 80),
                pad=rng.randrange(0, 8), dt=rng.choice((16, 20)) if D == 64 else rng.choice((16, 44)), dy=0, rms=rng.random() < 0.5,
                type=rng.choice(("bf16", "bf16", "f32")))
    case["dy"] = (D - case["dt"]) // 2 // 2 * 2
    while work(case)["bytes"] > 1.4e9:
        case["T"], case["Y"] = max(1, case["T"] - 1), max(2, case["Y"] * 7 // 8)
    return case


def _draw_states(rng, kind):
    H, D = rng.choice(((24, 128), (48, 64), (3, 64), (7, 128)))
    case = dict(kind=kind, B=rng.choice((1, 2)), S=_log_int(rng, 40, 7000), H=H, D=D, code=rng.choice(tuple(CODES)))
    if kind == "quantize":
        return dict(case, type=rng.choice(tuple(TYPES)))
    return dict(case, cached=rng.randrange(1, 9), fresh=rng.randrange(0, 3), to=rng.choice(("f32", "bf16", "code")))


def draw(rng):
    kind = rng.choice(("window", "window", "rope", "rope", "quantize", "merge"))
    return _draw_window(rng) if kind == "window" else _draw_rope(rng) if kind == "rope" else _draw_states(rng, kind)


# ------------------------------------------------------------------------------------------------ the work
def _visible_sums(Sq, Sk, left, right, sinks):
    """(pairs of a query and a key it sees, keys that some query sees); the queries are the last Sq of Sk positions."""
    p = torch.arange(Sk - Sq, Sk, dtype=torch.int64)
    lo, hi = (p - left).clamp(min=0), (p + right + 1).clamp(max=Sk)
    pairs = (hi - lo) + torch.minimum(lo.clamp(max=sinks), hi)
    first = int(lo[0])
    return int(pairs.sum()), int(hi[-1]) - first + min(first, sinks)


def _lengths(case):
    """Keys of each sequence: all Sk, or spread evenly between half of them and all."""
    B, Sk = case["B"], case["Sk"]
    if not case["ragged"]:
        return [Sk] * B
    return [max(case["Sq"], Sk - i * (Sk // 2) // max(1, B - 1)) for i in range(B)]


def _tokens(case):
    return case["text"] + case["T"] * case["Y"] * case["X"] + case["pad"]


def work(case):
    kind = case["kind"]
    if kind == "window":
        pairs = keys = 0
        for n in _lengths(case):
            a, b = _visible_sums(case["Sq"], n, case["left"], case["right"], case["sinks"])
            pairs, keys = pairs + a, keys + b
        rows = case["B"] * case["Sq"] * case["H"]
        return {"bytes": rows * (4 * case["D"] + 4) + keys * case["Hk"] * case["D"] * 4, "flops": 4 * case["D"] * case["H"] * pairs}
    if kind == "rope":
        n = 2 * case["B"] * _tokens(case) * case["H"] * case["D"]         # values of queries and keys
        size = 2 if case["type"] == "bf16" else 4
        return {"bytes": n * size * (3 if case["grad"] else 2), "flops": n * (24 if case["grad"] else 12)}
    rows, D = case["B"] * case["S"] * case["H"], case["D"]
    if kind == "quantize":
        return {"bytes": rows * (D * ((2 if case["type"] == "bf16" else 4) + 2) + 1), "flops": 4 * rows * D}
    out = {"f32": 4 * D, "bf16": 2 * D, "code": 2 * D + 1}[case["to"]]
    return {"bytes": rows * (case["cached"] * (D + 5) + case["fresh"] * (4 * D + 4) + out + 4),
            "flops": 2 * rows * D * (case["cached"] + case["fresh"])}


# ------------------------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=F32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    state = dict(case)
    B, H, D = case["B"], case["H"], case["D"]
    if case["kind"] == "window":
        # normalised queries and keys, as the models have behind their q / k norms
        state["q"] = randn(B, case["Sq"], H, D, dtype=BF16)
        state["k"], state["v"] = (randn(B, case["Sk"], case["Hk"], D, dtype=BF16) for _ in range(2))
        state["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    elif case["kind"] == "rope":
        S, t = _tokens(case), TYPES[case["type"]]
        state["q"], state["k"] = (randn(B, S, H, D, dtype=t, scale=1.5) for _ in range(2))
        state["weights"] = [(1 + randn(D, scale=0.2)).to(t) for _ in range(2)]
        state["biases"] = [None if case["rms"] else randn(D, dtype=t, scale=0.2) for _ in range(2)]
        if case["grad"]:
            state["dq"], state["dk"] = (randn(B, S, H, D, dtype=t, scale=0.01) for _ in range(2))
    else:
        S = case["S"]
        if case["kind"] == "quantize":
            # an attention output: heads of different size
            state["x"] = (randn(B, S, H, D, scale=0.1) * torch.exp(randn(1, 1, H, 1))).to(TYPES[case["type"]])
        else:
            state["cached"] = [_quantize(randn(B, S, H, D, scale=0.1), case["code"]) + (5 + randn(B, S, H),) for _ in range(case["cached"])]
            state["fresh"] = [(randn(B, S, H, D, scale=0.1), 5 + randn(B, S, H)) for _ in range(case["fresh"])]
    return state


# ------------------------------------------------------------------------------------------------ the operators
def run(state):
    kind = state["kind"]
    if own:
        return _own(state)
    if kind == "window":
        return _window(state)
    if kind == "rope":
        return _rope_grad(state) if state["grad"] else _rope(state)
    if kind == "quantize":
        codes, exponents = _quantize(state["x"].float(), state["code"])
        return _dequantize(codes, exponents).to(BF16), exponents
    return _merge(state)


def _own(state):
    from ditango_b200 import ops
    kind = state["kind"]
    if kind == "window":
        return ops.flash_window(state["q"], state["k"], state["v"], left=state["left"], right=state["right"], sinks=state["sinks"],
                                seqlens_k=state["lens"], out_dtype=BF16)
    if kind == "rope":
        rope = ops.GridRope((state["T"], state["Y"], state["X"]), (state["dt"], state["dy"], state["D"] - state["dt"] - state["dy"]))
        norms = [(w, b, 1e-6) for w, b in zip(state["weights"], state["biases"])]
        if not state["grad"]:
            return ops.norm_rope_grid(state["q"], state["k"], *norms, rope, text_len=state["text"], rms=state["rms"])
        return _present(ops.norm_rope_grid_backward(state["dq"], state["dk"], state["q"], state["k"], *norms, rope,
                                                    text_len=state["text"], rms=state["rms"]))
    if kind == "quantize":
        rows = ops.quantize_rows(state["x"], CODES[state["code"]])
        return ops.dequantize_rows(rows, BF16), rows.exponents
    states = [(o, l, ops.LSE_BSH) for o, l in state["fresh"]] + \
             [(ops.QuantizedRows(c, e), l, ops.LSE_BSH) for c, e, l in state["cached"]]
    if state["to"] == "f32":
        return ops.merge_states(states)
    if state["to"] == "bf16":
        out = torch.empty(state["B"], state["S"], state["H"], state["D"], dtype=BF16, device="cuda")
        return ops.merge_states(states, out_bf16=out, fp32_out=False)
    rows, lse = ops.merge_states(states, out_rows=CODES[state["code"]], fp32_out=False)
    return ops.dequantize_rows(rows, BF16), rows.exponents, lse


def _present(outputs):
    return tuple(x for x in outputs if x is not None)


# -- attention: blocks of queries against the keys that their window can reach, the first tokens beside them
BLOCK = 256


def _window(s):
    q, k, v, sinks, left, right = s["q"], s["k"], s["v"], s["sinks"], s["left"], s["right"]
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    dev = q.device
    lens = torch.full((B,), Sk, device=dev) if s["lens"] is None else s["lens"].long()
    rows = min(BLOCK, Sq)
    n = -(-Sq // rows)
    span = min(Sk, rows + left + right)
    at = (lens - Sq)[:, None] + torch.arange(n * rows, device=dev)                            # positions of the queries
    start = (at[:, ::rows] - left).clamp(min=0).clamp(max=Sk - span)                          # [B, n]
    window = start[:, :, None] + torch.arange(span, device=dev)                               # [B, n, span]
    first = torch.arange(min(sinks, Sk), device=dev).expand(B, n, -1)
    key = torch.cat([first, window], dim=2)
    of = torch.arange(B, device=dev)[:, None, None]
    kk, vv = (x[of, key].float().permute(0, 3, 1, 2, 4) for x in (k, v))                      # [B, Hk, n, keys, D]
    qq = torch.nn.functional.pad(q.float(), (0, 0, 0, 0, 0, n * rows - Sq))
    qq = qq.view(B, n, rows, Hk, H // Hk, D).permute(0, 3, 1, 4, 2, 5).reshape(B, Hk, n, -1, D)
    p = (qq @ kk.transpose(-1, -2)).mul_(1 / math.sqrt(D)).view(B, Hk, n, H // Hk, rows, -1)
    pos = at.view(B, n, rows)[..., None]
    j = key[:, :, None, :]
    is_first = (torch.arange(key.shape[2], device=dev) < first.shape[2])
    seen = (j <= pos + right) & (j < lens[:, None, None, None]) & torch.where(is_first, j < sinks, (j >= pos - left) & (j >= sinks))
    p.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, Hk, n, -1, p.shape[-1]) @ vv).view(B, Hk, n, H // Hk, rows, D) / total.masked_fill(total == 0, 1.0)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 2, 4, 1, 3, 5).reshape(B, n * rows, H, D)[:, :Sq]
    lse = lse.permute(0, 1, 3, 2, 4).reshape(B, H, n * rows)[:, :, :Sq]
    return out.to(BF16), lse.contiguous()


# -- norm and rotary positions
def _rotation(s, device):
    """cos and sin [tokens, D / 2] of the pairs' angles: 1 and 0 at the text, 0 and 0 behind the grid's last position."""
    axes = torch.cat([torch.full((d // 2,), i) for i, d in enumerate((s["dt"], s["dy"], s["D"] - s["dt"] - s["dy"]))])
    freq = torch.cat([10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d in (s["dt"], s["dy"], s["D"] - s["dt"] - s["dy"])])
    n = torch.arange(s["T"] * s["Y"] * s["X"], device=device)
    pos = torch.stack([n // (s["Y"] * s["X"]), n // s["X"] % s["Y"], n % s["X"]], dim=1).double()
    angle = pos[:, axes.to(device)] * freq.to(device)
    text, pad = angle.new_ones(s["text"], angle.shape[1]), angle.new_zeros(s["pad"], angle.shape[1])
    cos, sin = torch.cat([text, angle.cos(), pad]), torch.cat([0 * text, angle.sin(), pad])
    return cos.float()[None, :, None], sin.float()[None, :, None]


def _standard(x, rms):
    """(x normalised, 1 / its deviation)."""
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    scale = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    return x * scale, scale


def _rope(s):
    cos, sin = _rotation(s, s["q"].device)
    return _rope_one(s["q"], s["weights"][0], s["biases"][0], cos, sin, s["rms"]), _rope_one(s["k"], s["weights"][1], s["biases"][1], cos, sin, s["rms"])


def _rope_one(x, w, b, cos, sin, rms):
    y = _standard(x.float(), rms)[0] * w.float()
    y = y if b is None else y + b.float()
    re, im = y[..., 0::2], y[..., 1::2]
    return torch.stack([re * cos - im * sin, im * cos + re * sin], dim=-1).flatten(-2).to(x.dtype)


def _rope_grad(s):
    cos, sin = _rotation(s, s["q"].device)
    one = _rope_grad_one(s["dq"], s["q"], s["weights"][0], cos, sin, s["rms"])
    two = _rope_grad_one(s["dk"], s["k"], s["weights"][1], cos, sin, s["rms"])
    return _present((one[0], two[0], one[1], one[2], two[1], two[2]))


def _rope_grad_one(dz, x, w, cos, sin, rms):
    re, im = dz.float()[..., 0::2], dz.float()[..., 1::2]
    dy = torch.stack([re * cos + im * sin, im * cos - re * sin], dim=-1).flatten(-2)
    xs, scale = _standard(x.float(), rms)
    g = dy * w.float()
    inner = g - xs * (g * xs).mean(-1, keepdim=True)
    dx = scale * (inner if rms else inner - g.mean(-1, keepdim=True))
    return dx.to(x.dtype), (dy * xs).sum((0, 1, 2)).to(w.dtype), None if rms else dy.sum((0, 1, 2)).to(w.dtype)


# -- states in 8 bits: one power of two per row, the smallest that keeps its largest value within the codes
def _quantize(x, code):
    bits = x.abs().amax(-1).view(torch.int32)
    mantissa = {"int8": 0x7E0000, "e4m3": 0x600000}[code]           # of the largest code: 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
    b = ((bits + (0x7FFFFF - mantissa)) >> 23) - {"int8": 6, "e4m3": 8}[code]
    b = b.clamp(min=SMALLEST_EXPONENT)
    scaled = x * ((254 - b) << 23).view(F32)[..., None]
    codes = scaled.round().to(torch.int8) if code == "int8" else scaled.to(torch.float8_e4m3fn)
    return codes, b.to(torch.uint8)


def _dequantize(codes, exponents):
    return codes.float() * (exponents.int() << 23).view(F32)[..., None]


def _merge(s):
    values = torch.stack([o for o, _ in s["fresh"]] + [_dequantize(c, e) for c, e, _ in s["cached"]])
    lses = torch.stack([l for _, l in s["fresh"]] + [l for _, _, l in s["cached"]])
    top = lses.amax(0)
    weights = (lses - top).exp()
    total = weights.sum(0)
    out = (values * weights[..., None]).sum(0) / total[..., None]
    lse = top + total.log()
    if s["to"] != "code":
        return out.to(TYPES[s["to"]]), lse
    codes, exponents = _quantize(out, s["code"])
    return _dequantize(codes, exponents).to(BF16), exponents, lse


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "window":
        return _exact_window(s)
    if case["kind"] == "rope":
        return _exact_rope(s)
    if case["kind"] == "quantize":
        return _exact_rows(s["x"].double(), case["code"]), None
    logs = [l.double() for _, l in s["fresh"]] + [l.double() for _, _, l in s["cached"]]
    lse = torch.logsumexp(torch.stack(logs), 0)
    out = 0
    for i, (o, _) in enumerate(s["fresh"]):
        out = out + o.double() * (logs[i] - lse).exp()[..., None]
    for i, (c, e, _) in enumerate(s["cached"]):
        out = out + c.double() * _two_to(e.int() - 127)[..., None] * (logs[len(s["fresh"]) + i] - lse).exp()[..., None]
    return (out, lse) if case["to"] != "code" else (_exact_rows(out, case["code"]), None, lse)


def _two_to(n):
    return ((n.long() + 1023) << 52).view(torch.float64)


def _exact_rows(x, code):
    top = x.abs().amax(-1, keepdim=True)
    part, exponent = torch.frexp((top / LARGEST[code]).clamp(min=2.0 ** (SMALLEST_EXPONENT - 127)))
    exponent = exponent - (part == 0.5).int()            # the next whole exponent from below 2^exponent
    y = x * _two_to(-exponent)
    if code == "e4m3":             # three bits behind the leading one, the smallest step 2^-9
        step = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4
        y = torch.round(y * _two_to(-step)) * _two_to(step)
    else:
        y = torch.round(y)
    return y * _two_to(exponent)


def _exact_window(s):
    q, k, v = s["q"], s["k"], s["v"]
    B, Sq, H, D = q.shape
    group = H // k.shape[2]
    out, lse = q.new_zeros(q.shape, dtype=torch.float64), q.new_zeros(B, H, Sq, dtype=torch.float64)
    for b, length in enumerate(_lengths(s)):
        for i in range(0, Sq, 512):
            p = torch.arange(i, min(Sq, i + 512), device=q.device) + length - Sq
            j = torch.arange(length, device=q.device)
            keep = (j <= p[-1] + s["right"]) & ((j >= p[0] - s["left"]) | (j < s["sinks"]))
            j = j[keep]
            kk, vv = (x[b, :length][keep].double().repeat_interleave(group, dim=1).transpose(0, 1) for x in (k, v))
            score = q[b, i:i + 512].double().transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(D)
            hidden = (j[None] > p[:, None] + s["right"]) | ((j[None] < p[:, None] - s["left"]) & (j[None] >= s["sinks"]))
            score = score.masked_fill(hidden, -math.inf)
            lse[b, :, i:i + 512] = torch.logsumexp(score, -1)
            out[b, i:i + 512] = (torch.softmax(score, -1) @ vv).transpose(0, 1)
    return out, lse


def _exact_rope(s):
    """By complex numbers; gradients by automatic differentiation."""
    grad = s["grad"]
    sizes = (s["dt"], s["dy"], s["D"] - s["dt"] - s["dy"])
    dev = s["q"].device
    grid = torch.meshgrid(*(torch.arange(m, dtype=torch.float64, device=dev) for m in (s["T"], s["Y"], s["X"])), indexing="ij")
    angle = torch.cat([p.reshape(-1, 1) / 10000.0 ** (torch.arange(d // 2, dtype=torch.float64, device=dev) * 2 / d) for p, d in zip(grid, sizes)], dim=1)
    turn = torch.polar(torch.ones_like(angle), angle)
    turn = torch.cat([turn.new_ones(s["text"], turn.shape[1]), turn, turn.new_zeros(s["pad"], turn.shape[1])])
    outs, grads = [], []
    for name, w, b in zip(("q", "k"), s["weights"], s["biases"]):
        leaves = [x.double().requires_grad_(grad) for x in (s[name], w) + (() if b is None else (b,))]
        x = leaves[0]
        if s["rms"]:
            y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * leaves[1]
        else:
            y = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-6) * leaves[1] + leaves[2]
        z = torch.view_as_real(torch.view_as_complex(y.unflatten(-1, (-1, 2))) * turn[None, :, None]).flatten(-2)
        outs.append(z)
        if grad:
            grads.append(torch.autograd.grad(z, leaves, s["d" + name].double()))
    if not grad:
        return tuple(outs)
    return (grads[0][0], grads[1][0]) + tuple(grads[0][1:]) + tuple(grads[1][1:])
