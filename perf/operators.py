"""The operators of a decode step with quantised weights and a quantised cache, as measured cases.

Three operators that run one after the other in every layer of such a step:

  dot      out[m, n] = sum_k x[m, k] * (w[n, k] - z[n, k / G]) * s[n, k / G] + bias[n], w in 4 bits, one scale per
           group of G values along k (u4 weights carry a zero point per group, s4 weights do not)
  append   new keys and values are rounded to 8 bits and stored in their pages of the cache; a page holds `page`
           tokens and has one scale for each head.  The scale is the least power of two at which the largest new
           value fits the type, and at least the page's scale before; where it grows, the page's earlier codes are
           rounded to it again
  attend   softmax(scale * q k^T) v over the pages, causal from the end of each sequence, optionally in a window

`prepare` makes the inputs, `run` is one call.  `own` selects the kernels; without it `run` computes the same in plain
torch operations in 32 bits."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2, "s8": torch.int8}
QMAX = {"e4m3": 448.0, "e5m2": 57344.0, "s8": 127.0}
# QMAX = fraction * 2^exponent, the fraction in [0.5, 1)
QMAX_PARTS = {"e4m3": (0.875, 9), "e5m2": (0.875, 16), "s8": (127.0 / 128.0, 7)}


def listed():
    return [
        # A small projection for one token: latency.
        dict(name="dot small", op="dot", m=1, n=1024, k=2048, group=64, type="f16", zeros=False, bias=True),
        # The up projection of a large MLP for one token: the weights are streamed once.
        dict(name="dot one token", op="dot", m=1, n=28672, k=8192, group=128, type="bf16", zeros=False, bias=False),
        # The down projection for a batch of sixteen, with zero points.
        dict(name="dot sixteen", op="dot", m=16, n=8192, k=28672, group=128, type="bf16", zeros=True, bias=False),
        # Sizes that divide by nothing large, small groups, a few drafted tokens.
        dict(name="dot ragged", op="dot", m=5, n=5003, k=4416, group=32, type="f16", zeros=True, bias=True),
        # One short sequence, heads of 64: latency.
        dict(name="attend small", op="attend", batch=1, new=1, heads=8, kv_heads=2, dim=64, page=16, lo=37, hi=37, code="e4m3", type="f16", window=0, ragged=False, lse=False),
        # An ordinary serving batch with lengths all over the range and an idle slot.
        dict(name="attend batch", op="attend", batch=32, new=1, heads=32, kv_heads=8, dim=128, page=64, lo=0, hi=4096, code="e4m3", type="bf16", window=0, ragged=False, lse=False),
        # Two very long contexts: the work of one sequence has to be spread over the whole card.
        dict(name="attend long", op="attend", batch=2, new=1, heads=64, kv_heads=8, dim=128, page=128, lo=100003, hi=131072, code="e5m2", type="bf16", window=0, ragged=False, lse=True),
        # Drafted tokens checked together, some slots with fewer of them.
        dict(name="attend drafts", op="attend", batch=16, new=5, heads=32, kv_heads=4, dim=128, page=32, lo=5, hi=8191, code="s8", type="bf16", window=0, ragged=True, lse=True),
        # Wide heads, one key head, a sliding window.
        dict(name="attend window", op="attend", batch=7, new=1, heads=6, kv_heads=1, dim=256, page=16, lo=700, hi=20011, code="e4m3", type="f16", window=1000, ragged=False, lse=False),
        # One new token for each of a few sequences, 8-bit integers: latency.
        dict(name="append small", op="append", batch=3, new=1, kv_heads=2, dim=64, page=16, lo=1, hi=90, code="s8", type="f16", ragged=False),
        # One new token for each sequence of a serving batch.
        dict(name="append batch", op="append", batch=64, new=1, kv_heads=8, dim=128, page=64, lo=1, hi=2000, code="e4m3", type="bf16", ragged=False),
        # Whole prompts of different lengths behind shared starts.
        dict(name="append prompts", op="append", batch=8, new=4096, kv_heads=8, dim=128, page=64, lo=0, hi=1000, code="e4m3", type="bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("dot", "attend", "append"))
    if op == "dot":
        m, group = _log(rng, 1, 32), rng.choice((32, 64, 128))
        k = group * max(2, _log(rng, 512, 28672) // group)
        n = min(_log(rng, 256, 28672), 235_000_000 // k)
        zeros = rng.random() < 0.5
        return dict(op=op, m=m, n=n, k=k, group=group, type=rng.choice(("bf16", "f16")), zeros=zeros, bias=rng.random() < 0.5)
    kv_heads, dim, page = rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 96, 128, 128, 256)), rng.choice((16, 32, 64, 128))
    code, kind = rng.choice(("e4m3", "e4m3", "e5m2", "s8")), rng.choice(("bf16", "bf16", "f16"))
    batch = _log(rng, 1, 64)
    if op == "attend":
        new = rng.choice((1, 1, 1, 2, 3, 5, 8))
        hi = max(new + 1, min(_log(rng, 16, 131072), 250_000_000 // (batch * kv_heads * dim)))
        lo = rng.choice((0, hi, rng.randrange(new, hi)))
        return dict(op=op, batch=batch, new=new, heads=kv_heads * rng.choice((1, 2, 4, 5, 8)), kv_heads=kv_heads, dim=dim, page=page, lo=lo, hi=hi, code=code, type=kind,
                    window=rng.choice((0, 0, 0, _log(rng, 1, 4096))), ragged=new > 1 and rng.random() < 0.5, lse=rng.random() < 0.5)
    new = rng.choice((1, 1, rng.randrange(2, 9), _log(rng, 9, 4096)))
    hi = _log(rng, 1, 4000)
    new = max(1, min(new, 32_000_000 // (batch * kv_heads * dim)))
    hi = max(1, min(hi, 100_000_000 // (batch * kv_heads * dim)))
    return dict(op=op, batch=batch, new=new, kv_heads=kv_heads, dim=dim, page=page, lo=rng.randrange(0, hi + 1), hi=hi, code=code, type=kind, ragged=new > 1 and rng.random() < 0.5)


def _spread(lo, hi, count):
    return [hi] if count == 1 else [lo + (hi - lo) * i // (count - 1) for i in range(count)]


def _lengths(case):
    """(tokens before the call, new tokens) of each sequence: the lengths from lo to hi in even steps."""
    batch, new = case["batch"], case["new"]
    fresh = [max(1, new - (i * new) // (batch + 1)) if case["ragged"] else new for i in range(batch)]
    if case["op"] == "append":
        return _spread(case["lo"], case["hi"], batch), fresh
    total = _spread(case["lo"], case["hi"], batch)
    fresh = [min(f, t) for f, t in zip(fresh, total)]  # an idle slot has no token at all
    return [t - f for t, f in zip(total, fresh)], fresh


def _codes(shape, code, gen):
    if code == "s8":
        return torch.randint(-127, 128, shape, device="cuda", generator=gen, dtype=torch.int8)
    x = torch.randn(shape, device="cuda", generator=gen, dtype=torch.bfloat16)
    return x.mul_(QMAX[code] / 6).clamp_(-QMAX[code], QMAX[code]).to(CODES[code])


def _table(lens, page, gen):
    """Pages of the sequences in random places of the cache; entries behind a sequence's last page are -1."""
    counts = (lens + page - 1) // page
    total = int(counts.sum())
    width = max(1, int(counts.max()))
    perm = torch.randperm(total + 3, device="cuda", generator=gen).to(torch.int32)
    first = torch.cumsum(counts, 0) - counts
    at = torch.arange(width, device="cuda")
    inside = at[None, :] < counts[:, None]
    return torch.where(inside, perm[torch.where(inside, first[:, None] + at[None, :], 0)], -1).to(torch.int32).contiguous(), total + 3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    kind = DTYPES[case["type"]]
    s = dict(case)
    if case["op"] == "dot":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        s["x"] = rand((m, k)).to(kind)
        s["w"] = torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen, dtype=torch.uint8)
        s["scale"] = ((torch.rand((n, k // g), device="cuda", generator=gen) + 0.5) * (0.3 / math.sqrt(k))).to(kind)
        s["zero"] = torch.randint(5, 11, (n, k // g), device="cuda", generator=gen, dtype=torch.uint8) if case["zeros"] else None
        s["bias"] = rand((n,)).to(kind) if case["bias"] else None
        if own:
            import xla_b200

            s["out"] = torch.empty((m, n), dtype=kind, device="cuda")
            s["call"] = xla_b200.DotW4Call([s["x"], s["w"], s["scale"]] + [s[p] for p in ("zero", "bias") if s[p] is not None], [s["out"]],
                                           weight_type=xla_b200.U4 if case["zeros"] else xla_b200.S4, bias=case["bias"])
    else:
        before, fresh = (torch.tensor(v, device="cuda") for v in _lengths(case))
        order = torch.randperm(case["batch"], device="cuda", generator=gen)
        before, fresh = before[order], fresh[order]
        batch, new, kvh, dim, page, code = (case[p] for p in ("batch", "new", "kv_heads", "dim", "page", "code"))
        s["table"], pages = _table(before + fresh, page, gen)
        s["lens"], s["fresh"] = (before + fresh).to(torch.int32), fresh.to(torch.int32)
        for p in ("k", "v"):
            s[p] = _codes((pages, kvh, page, dim), code, gen)
            s[p + "_scale"] = (torch.rand((pages, kvh), device="cuda", generator=gen) * 1.5 + 0.5) * (3.0 / QMAX[code])
            if case["op"] == "append":  # scales as an earlier append left them
                s[p + "_scale"] = torch.exp2(torch.floor(torch.log2(s[p + "_scale"])))
                s[p + "_new"] = (rand((batch, new, kvh, dim)) * (0.25 + torch.rand((batch, new, kvh, 1), device="cuda", generator=gen))).to(kind)
        cache = [s["k"], s["v"], s["k_scale"], s["v_scale"]]
        more = [s["fresh"]] if case["ragged"] or (case["op"] == "attend" and case["lo"] < new) else []
        if case["op"] == "attend":
            s["q"] = (rand((batch, new, case["heads"], dim)) * 2).to(kind)
        if own:
            import xla_b200

            if case["op"] == "attend":
                s["out"] = torch.empty_like(s["q"])
                s["lse_out"] = torch.empty((batch, new, case["heads"]), dtype=torch.float32, device="cuda") if case["lse"] else None
                s["work"] = torch.empty(xla_b200.paged_attention_workspace_bytes(batch, new, case["heads"], kvh, dim), dtype=torch.int8, device="cuda")
                s["call"] = xla_b200.PagedAttentionKv8Call([s["q"]] + cache + [s["table"], s["lens"]] + more, [s["out"]] + ([s["lse_out"]] if case["lse"] else []) + [s["work"]],
                                                           softmax_scale=dim ** -0.5, window=case["window"], emit_lse=case["lse"])
            else:
                s["call"] = xla_b200.KvCacheAppendCall([s["k_new"], s["v_new"]] + cache + [s["table"], s["lens"]] + more, cache)
    if own:
        s["call"].instantiate()
    return s


def run(s):
    if own:
        s["call"].execute(torch.cuda.current_stream().cuda_stream, 0)
        if s["op"] == "dot":
            return {"out": s["out"]}
        if s["op"] == "attend":
            return {"out": s["out"], "lse": s["lse_out"]} if s["lse"] else {"out": s["out"]}
        return {p: s[p] for p in ("k", "v", "k_scale", "v_scale")}
    return {"dot": _dot, "attend": _attend, "append": _append}[s["op"]](s)


def _take(codes, at):
    return codes.view(torch.uint8)[at].view(codes.dtype)


def _dot(s):
    n, k, g = s["n"], s["k"], s["group"]
    w = torch.stack((s["w"] & 15, s["w"] >> 4), dim=-1).reshape(n, k // g, g).float()  # the even k in the low four bits
    w = w - s["zero"].float()[:, :, None] if s["zeros"] else torch.where(w > 7, w - 16, w)
    out = s["x"].float() @ (w * s["scale"].float()[:, :, None]).reshape(n, k).t()
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return {"out": out.to(s["x"].dtype)}


def _attend(s):
    batch, new, heads, dim = s["q"].shape
    kvh, page, table = s["kv_heads"], s["page"], s["table"].long()
    tokens = table.shape[1] * page
    at = torch.arange(tokens, device="cuda")
    used = at[None, :] < s["lens"][:, None]
    held = lambda p: (_take(s[p], table.clamp(min=0)).float() * s[p + "_scale"][table.clamp(min=0)][..., None, None]).transpose(1, 2).reshape(batch, kvh, tokens, dim)  # noqa: E731
    q = s["q"].float().reshape(batch, new, kvh, heads // kvh, dim).permute(0, 2, 3, 1, 4).reshape(batch, kvh, -1, dim)
    scores = (q @ held("k").transpose(2, 3)).reshape(batch, heads, new, tokens) * dim ** -0.5
    i = torch.arange(new, device="cuda")
    here = (s["lens"] - s["fresh"])[:, None] + i
    seen = used[:, None, :] & (at <= here[:, :, None]) & (i < s["fresh"][:, None])[:, :, None]
    if s["window"]:
        seen = seen & (at > here[:, :, None] - s["window"])
    scores = torch.where(seen[:, None], scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(used[:, None, :, None], held("v"), 0.0)
    out = (p.reshape(batch, kvh, -1, tokens) @ v).reshape(batch, heads, new, dim) / torch.where(total == 0, 1.0, total)
    answer = {"out": out.transpose(1, 2).to(s["q"].dtype)}
    if s["lse"]:
        answer["lse"] = (torch.log(total) + torch.where(top == -torch.inf, 0.0, top))[..., 0].transpose(1, 2).contiguous()
    return answer


def _append(s):
    batch, new, kvh, dim = s["k_new"].shape
    page, table, code = s["page"], s["table"].long(), s["code"]
    fraction, exponent = QMAX_PARTS[code]
    start = (s["lens"] - s["fresh"]).long()
    blocks = torch.arange((new - 1) // page + 2, device="cuda")
    index = start[:, None] // page + blocks  # the pages that new tokens reach
    at = index[:, :, None] * page + torch.arange(page, device="cuda")  # positions, [batch, blocks, page]
    i = at - start[:, None, None]
    fresh, old = (i >= 0) & (i < s["fresh"][:, None, None]), i < 0
    written = fresh.any(-1)
    where = torch.where(written, torch.gather(table, 1, index.clamp(max=table.shape[1] - 1)), 0)
    here = torch.arange(batch, device="cuda")[:, None, None]
    target = where[written]

    def store(codes, scales, values):
        x = values[here, i.clamp(0, new - 1)].transpose(2, 3).float()  # [batch, blocks, kv_heads, page, dim]
        x = torch.where(fresh[:, :, None, :, None], x, 0.0)
        part, power = torch.frexp(x.abs().amax((-1, -2)))
        power = torch.where(part == 0, -126, torch.clamp(power - exponent + (part > fraction), min=-126))
        before = torch.where(old.any(-1)[:, :, None], scales[where], 0.0)
        scale = torch.maximum(before, ((power + 127) << 23).view(torch.float32))
        held = _take(codes, where)
        y = torch.where(fresh[:, :, None, :, None], x, held.float() * before[..., None, None]) / scale[..., None, None]
        y = torch.clamp(y, -QMAX[code], QMAX[code])
        y = torch.round(y).to(torch.int8) if code == "s8" else y.to(CODES[code])
        y = torch.where((fresh | old)[:, :, None, :, None], y.view(torch.uint8), held.view(torch.uint8))
        codes.view(torch.uint8)[target] = y[written]
        scales[target] = scale[written]

    store(s["k"], s["k_scale"], s["k_new"])
    store(s["v"], s["v_scale"], s["v_new"])
    return {p: s[p] for p in ("k", "v", "k_scale", "v_scale")}


def _seen(case):
    """Tokens that some query of the sequence sees, summed over the sequences, and the pairs of query and token."""
    tokens = pairs = 0
    for before, fresh in zip(*_lengths(case)):
        sees = [min(before + i + 1, case["window"] or before + i + 1) for i in range(fresh)]
        tokens += min(before + fresh, sees[-1] + fresh - 1) if sees else 0
        pairs += sum(sees)
    return tokens, pairs


def work(case):
    size = torch.finfo(DTYPES[case["type"]]).bits // 8
    if case["op"] == "dot":
        m, n, k, g = (case[p] for p in ("m", "n", "k", "group"))
        return {"bytes": n * k // 2 + n * (k // g) * (size + case["zeros"]) + size * (m * k + m * n + n * case["bias"]), "flops": 2 * m * n * k}
    batch, new, kvh, dim, page = (case[p] for p in ("batch", "new", "kv_heads", "dim", "page"))
    if case["op"] == "attend":
        tokens, pairs = _seen(case)
        moved = 2 * tokens * kvh * dim + 8 * (tokens // page) * kvh + batch * new * case["heads"] * (2 * dim * size + 4 * case["lse"])
        return {"bytes": moved, "flops": 4 * pairs * case["heads"] * dim}
    before, fresh = _lengths(case)
    pages = sum((b + f - 1) // page - b // page + 1 for b, f in zip(before, fresh))
    return {"bytes": 2 * (sum(fresh) * kvh * dim * (size + 1) + 8 * pages * kvh), "flops": 2 * sum(fresh) * kvh * dim * 4}


def exact(case, seed):
    state = prepare(case, seed)
    return {"dot": _exact_dot, "attend": _exact_attend, "append": _exact_append}[case["op"]](case, state)


def _exact_dot(case, s):
    values = torch.arange(256, device="cuda")
    nibbles = torch.stack((values % 16, values // 16), 1).double()
    if not case["zeros"]:
        nibbles = (nibbles + 8) % 16 - 8
    x, out = s["x"].double(), []
    for rows in range(0, case["n"], 2048):
        part = slice(rows, rows + 2048)
        w = nibbles[s["w"][part].int()].reshape(-1, case["k"] // case["group"], case["group"])
        if case["zeros"]:
            w = w - s["zero"][part].double().unsqueeze(2)
        w = w * s["scale"][part].double().unsqueeze(2)
        out.append(torch.matmul(w.reshape(w.shape[0], -1), x.t()).t() + (s["bias"][part].double() if case["bias"] else 0.0))
    return {"out": torch.cat(out, 1)}


def _exact_attend(case, s):
    kvh, dim, share = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:3], -torch.inf, dtype=torch.float64, device="cuda")
    lens, fresh = s["lens"].tolist(), s["fresh"].tolist()
    for b, (length, count) in enumerate(zip(lens, fresh)):
        pages = s["table"][b, : -(-length // case["page"])].long()
        for h in range(kvh):
            if not count:
                continue
            k, v = ((_take(s[p], (pages, h)).double() * s[p + "_scale"][pages, h].double()[:, None, None]).reshape(-1, dim)[:length] for p in ("k", "v"))
            for i in range(count):
                last = length - count + i + 1
                first = max(0, last - case["window"]) if case["window"] else 0
                scores = s["q"][b, i, h * share : (h + 1) * share].double() @ k[first:last].t() / math.sqrt(dim)
                lse[b, i, h * share : (h + 1) * share] = torch.logsumexp(scores, 1)
                out[b, i, h * share : (h + 1) * share] = torch.softmax(scores, 1) @ v[first:last]
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_append(case, s):
    code, page = case["code"], case["page"]
    bits, least = {"e4m3": (3, -6), "e5m2": (2, -14), "s8": (0, 0)}[code]

    def rounded(y):
        step = torch.ones_like(y)
        if code != "s8":
            step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.where(y == 0, 1.0, y.abs()))), min=least) - bits)
        return torch.clamp(torch.round(y / step) * step, -QMAX[code], QMAX[code])

    answer = {p: s[p].double() for p in ("k", "v", "k_scale", "v_scale")}
    for b, (length, count) in enumerate(zip(s["lens"].tolist(), s["fresh"].tolist())):
        begin = length - count
        for j in range(begin // page, -(-length // page)):
            at, first, last = int(s["table"][b, j]), max(begin, j * page), min(length, (j + 1) * page)
            for p in ("k", "v"):
                x = s[p + "_new"][b, first - begin : last - begin].double().transpose(0, 1)
                top = x.abs().amax((1, 2)) / QMAX[code]
                part, power = torch.frexp(top)
                scale = torch.exp2(torch.clamp(power.double() - (part == 0.5).double(), min=-126.0))
                if first > j * page:
                    scale = torch.maximum(scale, answer[p + "_scale"][at])
                    held = answer[p][at, :, : first - j * page]
                    answer[p][at, :, : first - j * page] = rounded(held * (answer[p + "_scale"][at] / scale)[:, None, None])
                answer[p][at, :, first - j * page : last - j * page] = rounded(x / scale[:, None, None])
                answer[p + "_scale"][at] = scale
    return answer if code != "s8" else {**answer, "k": None, "v": None}
