"""Keys and values of streams that are kept in pages, as cases that can be timed and compared.

  extend    pages for the new tokens of each stream, and the slot of each of them (ops.extend_pages)
  release   pages that nothing needs any more go back (ops.release_pages)
  write     keys and values of new tokens into their slots (ops.write_pages)
  attend    attention of the streams' new tokens over their pages (ops.flash_paged)

With `own` false, `run` computes them by elementary torch operations, in 32 bits; with `own` true it calls the package.
"""
import math

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # Seven streams get a token each: what happens in front of every step of single tokens.  Latency is all there is.
        dict(name="extend_tokens", kind="extend", B=7, M=300, P=64, lo=1, hi=17000, new_lo=1, new_hi=1),
        # 256 streams get a latent frame of 1350 tokens (30 x 45) each.
        dict(name="extend_frames", kind="extend", B=256, M=400, P=64, lo=226, hi=17776, new_lo=1350, new_hi=1350),
        # 96 streams, windows of 5 frames of 1350 tokens: the frame behind each window goes, the 226 text tokens stay.
        dict(name="release_frames", kind="release", B=96, M=1200, P=16, lo=7000, hi=17776, keep=226, window=6750),
        # The keys and values of a token of each of 24 streams, 8 heads of 128, into small pages.
        dict(name="write_tokens", kind="write", T=24, Hk=8, D=128, P=16, spare=0),
        # Two streams' latent frames of 45 x 80 tokens, HunyuanVideo's heads; rows behind them are padding.
        dict(name="write_frames", kind="write", T=7219, Hk=24, D=128, P=128, spare=19),
        # One token of a short stream, four query heads to a key head, small pages.  The smallest attention.
        dict(name="attend_token", kind="attend", B=1, new_lo=1, new_hi=1, lo=1500, hi=1500, H=32, Hk=8, D=64, P=16, left=-1, right=0, sinks=0),
        # A token of each of 24 streams whose lengths differ by two orders of magnitude.
        dict(name="attend_tokens_ragged", kind="attend", B=24, new_lo=1, new_hi=1, lo=200, hi=30000, H=32, Hk=8, D=128, P=16, left=-1, right=0, sinks=0),
        # One token against HunyuanVideo's whole 720p sequence, a key head to each query head: the longest cache.
        dict(name="attend_token_hunyuan", kind="attend", B=1, new_lo=1, new_hi=1, lo=119056, hi=119056, H=24, Hk=24, D=128, P=128, left=-1, right=0, sinks=0),
        # Five drafted tokens of each of seven streams, eight query heads to a key head.
        dict(name="attend_drafts", kind="attend", B=7, new_lo=5, new_hi=5, lo=5003, hi=20011, H=32, Hk=4, D=64, P=32, left=-1, right=0, sinks=0),
        # Two streams' next latent frame (1350 tokens) against all of CogVideoX's frames so far and the text.
        dict(name="attend_frame_cogvideox", kind="attend", B=2, new_lo=1350, new_hi=1350, lo=11026, hi=17776, H=48, Hk=48, D=64, P=64, left=-1, right=-1, sinks=0),
        # The next frame of HunyuanVideo (3600 tokens), each token against the two frames before it, a frame behind it and the text.
        dict(name="attend_frame_hunyuan", kind="attend", B=1, new_lo=3600, new_hi=3600, lo=29764, hi=29764, H=24, Hk=24, D=128, P=128, left=7200, right=3599, sinks=256),
        # A batch as a server has it: single tokens beside chunks of prompts, causal.  The most work.
        dict(name="attend_mixed", kind="attend", B=9, new_lo=1, new_hi=2500, lo=2500, hi=20000, H=32, Hk=8, D=128, P=16, left=-1, right=0, sinks=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_attend(rng):
    Hk, group = rng.choice(((1, 8), (2, 16), (4, 8), (8, 4), (8, 1), (12, 2), (24, 1), (48, 1)))
    lo = rng.choice((_log_int(rng, 1, 60000), _log_int(rng, 1000, 60000)))
    hi = rng.choice((lo, _log_int(rng, lo, 60000)))
    new_hi = rng.choice((1, 1, _log_int(rng, 1, 16), _log_int(rng, 1, 200), _log_int(rng, 16, 4000)))
    right = rng.choice((0, 0, -1, _log_int(rng, 1, 4000)))
    case = dict(kind="attend", B=_log_int(rng, 1, 40), new_lo=rng.choice((new_hi, _log_int(rng, 1, new_hi))), new_hi=new_hi, lo=lo, hi=hi, H=Hk * group, Hk=Hk,
                D=rng.choice((64, 128)), P=rng.choice((16, 32, 64, 128, 256)), left=rng.choice((-1, -1, _log_int(rng, 16, 8000))), right=right,
                sinks=rng.choice((0, 0, _log_int(rng, 1, 300))))
    most = max(work(c)["flops"] for c in listed())
    while case["B"] > 1 and (work(case)["flops"] > most or _keys(case) * case["Hk"] * case["D"] > 3.6e8):
        case["B"] = case["B"] * 2 // 3
    while work(case)["flops"] > most or _keys(case) * case["Hk"] * case["D"] > 3.6e8:
        case["lo"], case["hi"] = max(1, case["lo"] * 3 // 4), max(1, case["hi"] * 3 // 4)
        case["new_hi"] = max(1, case["new_hi"] * 4 // 5)
        case["new_lo"] = min(case["new_lo"], case["new_hi"])
    return case


def draw(rng):
    kind = rng.choice(("extend", "release", "write", "attend", "attend", "attend", "attend"))
    if kind == "attend":
        return _draw_attend(rng)
    if kind == "write":
        T = _log_int(rng, 1, 7000)
        return dict(kind="write", T=T, Hk=rng.choice((1, 3, 4, 8, 24)), D=rng.choice((64, 128)), P=rng.choice((16, 32, 64, 128, 256)),
                    spare=rng.choice((0, rng.randrange(0, min(T, 40)))))
    P, hi = rng.choice((16, 32, 64, 128)), _log_int(rng, 100, 17000)
    case = dict(kind=kind, B=_log_int(rng, 1, 256), P=P, lo=_log_int(rng, 1, hi), hi=hi)
    if kind == "release":
        return dict(case, M=hi // P + 2, keep=rng.choice((0, rng.randrange(1, 300))), window=_log_int(rng, 16, 9000))
    new = rng.choice((1, _log_int(rng, 1, 1350)))
    return dict(case, M=(hi + new) // P + 2, new_lo=_log_int(rng, 1, new), new_hi=new)


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo, evenly over their logarithm, and not in order."""
    if n == 1:
        return [hi]
    values = [int(round(hi * (lo / hi) ** (i / (n - 1)))) for i in range(n)]
    step = next(s for s in (7, 5, 3, 2, 1) if math.gcd(s, n) == 1)
    return [values[i * step % n] for i in range(n)]


def _lengths(case):
    """(new tokens, tokens in all) of each stream."""
    new = _spread(case["new_lo"], case["new_hi"], case["B"])
    return list(zip(new, (max(a, b) for a, b in zip(new, _spread(case["lo"], case["hi"], case["B"])[::-1]))))


def _pages(tokens, P):
    return -(-tokens // P)


# ------------------------------------------------------------------------------------------------ the work
def _visible(case, n, total):
    """(pairs of a query and a key that it sees, keys that some query sees); the n queries are the last positions."""
    x = torch.arange(total - n, total, dtype=torch.int64)
    hi = (x + case["right"] + 1).clamp(max=total) if case["right"] >= 0 else torch.full_like(x, total)
    lo = (x - case["left"]).clamp(min=0) if case["left"] >= 0 else torch.zeros_like(x)
    pairs = hi - lo + torch.minimum(lo.clamp(max=case["sinks"]), hi)
    return int(pairs.sum()), int(hi[-1]) - int(lo[0]) + min(int(lo[0]), case["sinks"])


def _keys(case):
    return sum(total for _, total in _lengths(case))


def work(case):
    kind = case["kind"]
    if kind == "write":
        return {"bytes": (case["T"] - case["spare"]) * (case["Hk"] * case["D"] * 8 + 4), "flops": 0}
    if kind == "attend":
        pairs = keys = rows = 0
        for n, total in _lengths(case):
            a, b = _visible(case, n, total)
            pairs, keys, rows = pairs + a, keys + b, rows + n
        return {"bytes": rows * case["H"] * (case["D"] * 4 + 4) + keys * case["Hk"] * case["D"] * 4, "flops": 4 * case["D"] * case["H"] * pairs}
    P = case["P"]
    if kind == "extend":
        old, new = _cached(case), _spread(case["new_lo"], case["new_hi"], case["B"])
        pages = sum(_pages(a + n, P) - _pages(a, P) for a, n in zip(old, new))
        return {"bytes": 4 * (sum(new) + 2 * pages + 5 * case["B"]), "flops": 0}
    return {"bytes": 4 * (2 * case["B"] * case["M"] + 4 * case["B"]), "flops": 0}


def _cached(case):
    return _spread(case["lo"], case["hi"], case["B"])


# ------------------------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").int()

    def pages(number, Hk, P, D):
        """[number, P, Hk, D], the tokens of a page's head one after another in memory."""
        return torch.randn(number, Hk, P, D, generator=g, device="cuda", dtype=F32).to(BF16).transpose(1, 2)

    state = dict(case)
    kind, P = case["kind"], case["P"]
    if kind == "write":
        T, Hk, D = case["T"], case["Hk"], case["D"]
        number = _pages(T, P) * 5 // 4 + 1
        # (the last page is no part of the pool: the plain form puts padding there)
        state["k_all"], state["v_all"] = (pages(number + 1, Hk, P, D) for _ in range(2))
        state["k"], state["v"] = (torch.randn(T, Hk, D, generator=g, device="cuda").to(BF16) for _ in range(2))
        order = shuffled(number)
        t = torch.arange(T, device="cuda")
        state["slots"] = (order[t // P] * P + t % P).int()
        if case["spare"]:
            state["slots"][T - case["spare"]:] = -1
        return state
    if kind == "attend":
        lengths = _lengths(case)
        T, H, D = sum(n for n, _ in lengths), case["H"], case["D"]
        counts = [_pages(total, P) for _, total in lengths]
        number = sum(counts) + 3
        state["k"], state["v"] = (pages(number, case["Hk"], P, D) for _ in range(2))
        state["table"] = _table(shuffled(number), counts, max(counts) + 1)
        state["q"] = torch.randn(T, H, D, generator=g, device="cuda").to(BF16)
        state["lens"] = ints([total for _, total in lengths])
        state["cu"] = torch.cat([ints([0]), ints([n for n, _ in lengths]).cumsum(0).int()])
        return state
    counts = [_pages(n, P) for n in _cached(case)]
    if kind == "extend":
        new = _spread(case["new_lo"], case["new_hi"], case["B"])
        number = sum(counts) + sum(_pages(n, P) + 1 for n in new) + 5
        state["new"], state["tokens"] = ints(new), sum(new)
    else:
        number = sum(counts) + 5
        ends = [max(0, n - case["window"]) for n in _cached(case)]
        # (every third stream is over and gives all back)
        state["begin"] = ints([0 if i % 3 == 2 else case["keep"] for i in range(case["B"])])
        state["end"] = ints([n if i % 3 == 2 else e for i, (n, e) in enumerate(zip(_cached(case), ends))])
        state["new_table"] = torch.empty(case["B"], case["M"], dtype=torch.int32, device="cuda")
    order = shuffled(number)
    state["table"] = _table(order, counts, case["M"])
    state["lens"] = ints(_cached(case))
    state["free"] = torch.cat([order[sum(counts):], order[:sum(counts)]])          # (those in use lie above the count)
    state["count"] = ints([number - sum(counts)])
    return state


def _table(order, counts, columns):
    """Rows of page numbers, one stream's after another's, -1 behind a stream's last page."""
    n = torch.tensor(counts, device=order.device)
    j = torch.arange(columns, device=order.device)
    at = (n.cumsum(0) - n)[:, None] + j
    return torch.where(j < n[:, None], order[at.clamp(max=order.numel() - 1)], -1).int()


# ------------------------------------------------------------------------------------------------ the operators
def run(state):
    kind = state["kind"]
    if own:
        return _own(state)
    return {"extend": _extend, "release": _release, "write": _write, "attend": _attend}[kind](state)


def _own(s):
    from ditango_b200 import ops
    kind, P = s["kind"], s["P"]
    if kind == "extend":
        plan = ops.extend_pages(s["table"], s["lens"], s["new"], s["free"], s["count"], P, s["tokens"])
        return plan.slots, plan.cu_seqlens, plan.seqlens, s["table"], plan.free_count, plan.missing
    if kind == "release":
        left = ops.release_pages(s["table"], s["lens"], s["free"], s["count"], s["begin"], s["end"], P, out_table=s["new_table"])
        return s["new_table"], left.seqlens, s["free"], left.free_count
    if kind == "write":
        k, v = s["k_all"][:-1], s["v_all"][:-1]
        ops.write_pages(s["k"], s["v"], k, v, s["slots"])
        return k, v
    return ops.flash_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], left=s["left"], right=s["right"], sinks=s["sinks"], cu_seqlens_q=s["cu"],
                           max_seqlen_q=s["new_hi"], max_seqlen_k=max(s["hi"], s["new_hi"]), out_dtype=BF16)


def _extend(s):
    """(slots, offsets of the streams' new tokens, lengths, table, free pages, pages that were missing)"""
    table, P, free, B = s["table"], s["P"], s["free"], s["B"]
    M = table.shape[1]
    old, new, count = s["lens"].long(), s["new"].long(), s["count"].long()
    now = old + new
    first, last = (old + P - 1) // P, (now + P - 1) // P
    need = last - first
    before = need.cumsum(0) - need
    missing = (need.sum() - count).clamp(min=0)
    bad = (now > M * P).any() | (new.sum() > s["tokens"])
    refused = (missing > 0) | bad
    j = torch.arange(M, device=table.device)
    at = (count - 1 - before[:, None] - (j - first[:, None])).clamp(min=0, max=free.numel() - 1)
    fresh = (j >= first[:, None]) & (j < last[:, None]) & ~refused
    table.copy_(torch.where(fresh, free[at], table))
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0))
    t = torch.arange(s["tokens"], device=table.device)
    of = torch.searchsorted(cu, t, right=True) - 1
    inside = (of < B) & ~refused
    of = of.clamp(max=B - 1)
    x = old[of] + t - cu[of]
    slots = torch.where(inside, table[of, (x // P).clamp(max=M - 1)].long() * P + x % P, -1)
    return (slots.int(), torch.where(refused, 0, cu).int(), torch.where(refused, old, now).int(), table,
            torch.where(refused, count, count - need.sum()).int(), torch.where(bad, -1, missing).int().view(1))


def _release(s):
    """(table, lengths, free pages, how many)"""
    table, P, free = s["table"], s["P"], s["free"]
    old, begin, end = (s[n].long()[:, None] for n in ("lens", "begin", "end"))
    j = torch.arange(table.shape[1], device=table.device)
    goes = (j * P < old) & (j * P >= begin) & (((j + 1) * P <= end) | (end >= old)) & (begin < end) & (table >= 0)
    place = goes.flatten().cumsum(0).view(goes.shape) - 1 + s["count"].long()
    # (what stays is put into a place behind the list)
    longer = torch.cat([free, free[:1]])
    longer.index_put_((torch.where(goes, place, free.numel()),), table)
    free.copy_(longer[:-1])
    left = torch.where((end >= old) & (begin < old), begin, old)
    return torch.where(goes, -1, table), left[:, 0].int(), free, (s["count"] + goes.sum()).int()


def _write(s):
    at, P = s["slots"].long(), s["P"]
    s["k_all"][at // P, at % P] = s["k"]              # (-1: the last page)
    s["v_all"][at // P, at % P] = s["v"]
    return s["k_all"][:-1], s["v_all"][:-1]


BLOCK = 256


def _attend(s):
    """Blocks of queries against the first keys and the run of keys that some of them see."""
    q, table, P, D, Hk, left, right = s["q"], s["table"], s["P"], s["D"], s["Hk"], s["left"], s["right"]
    group = s["H"] // Hk
    outs, lses, begin = [], [], 0
    for b, (n, total) in enumerate(_lengths(s)):
        for i in range(begin, begin + n, BLOCK):
            rows = min(BLOCK, begin + n - i)
            x = total - n + i - begin + torch.arange(rows, device=q.device)
            x0 = total - n + i - begin
            lo = 0 if left < 0 else max(0, x0 - left)
            hi = total if right < 0 else min(total, x0 + rows + right)
            j = torch.cat([torch.arange(min(s["sinks"], lo), device=q.device), torch.arange(lo, hi, device=q.device)])
            page, at = table[b].long()[j // P], j % P
            k, v = (y[page, at].float().transpose(0, 1) for y in (s["k"], s["v"]))                     # [Hk, keys, D]
            y = q[i:i + rows].float().view(rows, Hk, group, D).permute(1, 2, 0, 3).reshape(Hk, group * rows, D)
            p = (y @ k.transpose(1, 2)).mul_(1 / math.sqrt(D)).view(Hk, group, rows, -1)
            seen = torch.ones(rows, j.numel(), dtype=torch.bool, device=q.device)
            if right >= 0:
                seen &= j <= x[:, None] + right
            if left >= 0:
                seen &= (j >= x[:, None] - left) | (j < s["sinks"])
            p.masked_fill_(~seen, -math.inf)
            top = p.amax(-1, keepdim=True)
            p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
            sums = p.sum(-1, keepdim=True)
            out = (p.view(Hk, group * rows, -1) @ v).view(Hk, group, rows, D) / sums.masked_fill(sums == 0, 1.0)
            outs.append(out.permute(2, 0, 1, 3).reshape(rows, s["H"], D).to(BF16))
            lses.append((top + sums.log()).view(s["H"], rows))
        begin += n
    return torch.cat(outs), torch.cat(lses, dim=1)


# ------------------------------------------------------------------------------------------------ from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return _exact_write(s)
    if case["kind"] == "attend":
        return _exact_attend(s)
    return _exact_extend(s) if case["kind"] == "extend" else _exact_release(s)


def _exact_extend(s):
    """A page after another, on the host."""
    P = s["P"]
    table, lens, new, free, count = (s[n].tolist() for n in ("table", "lens", "new", "free", "count"))
    stack, slots, cu = free[:count[0]], [], [0]
    for b, n in enumerate(new):
        for x in range(lens[b], lens[b] + n):
            if x % P == 0:
                table[b][x // P] = stack.pop()
            slots.append(table[b][x // P] * P + x % P)
        cu.append(cu[-1] + n)
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (slots, cu, [a + n for a, n in zip(lens, new)], table, [len(stack)], [0]))


def _exact_release(s):
    P = s["P"]
    table, lens, free, count, begin, end = (s[n].tolist() for n in ("table", "lens", "free", "count", "begin", "end"))
    used, left = count[0], []
    for b, n in enumerate(lens):
        for j in range(-(-n // P)):
            tokens = range(j * P, min(n, (j + 1) * P))
            whole = tokens[0] >= begin[b] and (tokens[-1] < end[b] if end[b] >= n else (j + 1) * P <= end[b])
            if whole and table[b][j] >= 0:
                free[used], table[b][j] = table[b][j], -1
                used += 1
        left.append(begin[b] if end[b] >= n and begin[b] < n else n)
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (table, left, free, [used]))


def _exact_write(s):
    out = []
    kept = (s["slots"] >= 0).nonzero()[:, 0]
    for pages, rows in ((s["k_all"], s["k"]), (s["v_all"], s["v"])):
        flat = pages[:-1].double().flatten(0, 1)
        flat[s["slots"][kept].long()] = rows[kept].double()
        out.append(flat.view(-1, *pages.shape[1:]))
    return tuple(out)


def _exact_attend(s):
    q, P, H, Hk, D = s["q"], s["P"], s["H"], s["Hk"], s["D"]
    out, lse = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(H, q.shape[0], dtype=torch.float64, device=q.device)
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    for b, length in enumerate(lens):
        used = s["table"][b, :_pages(length, P)].long()
        k, v = (x[used].flatten(0, 1)[:length] for x in (s["k"], s["v"]))
        position = torch.arange(length, device=q.device)
        for head in range(Hk):
            kk, vv = k[:, head].double(), v[:, head].double()
            heads = slice(head * (H // Hk), (head + 1) * (H // Hk))
            for i in range(cu[b], cu[b + 1], 1024):
                e = min(cu[b + 1], i + 1024)
                x = length - cu[b + 1] + torch.arange(i, e, device=q.device)[:, None]
                hidden = position > x + s["right"] if s["right"] >= 0 else torch.zeros(e - i, length, dtype=torch.bool, device=q.device)
                if s["left"] >= 0:
                    hidden = hidden | ((position < x - s["left"]) & (position >= s["sinks"]))
                score = torch.einsum("ihd,jd->hij", q[i:e, heads].double(), kk) / math.sqrt(D)
                score = score.masked_fill(hidden, -math.inf)
                lse[heads, i:e] = torch.logsumexp(score, -1)
                out[i:e, heads] = torch.einsum("hij,jd->ihd", torch.softmax(score, -1), vv)
    return out, lse
