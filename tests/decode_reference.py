"""Plain 64-bit forms of the decode-step operators, and inputs for their tests, on any device."""
import math

import torch

S8, E4M3, E5M2 = torch.int8, torch.float8_e4m3fn, torch.float8_e5m2
QMAX = {S8: 127.0, E4M3: 448.0, E5M2: 57344.0}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # relative


def take(codes, at):
    """codes[at], also for the float types that torch does not index."""
    return codes.view(torch.uint8)[at].view(codes.dtype)


def weights(w, zero, group):
    """The integers w - z that the bytes [n, k / 2] stand for, [n, k]."""
    q = torch.stack((w & 15, w >> 4), -1).flatten(1).double()
    if zero is None:
        return torch.where(q > 7, q - 16, q)
    return q - (zero & 15).double().repeat_interleave(group, 1)


def dot(x, w, scale, zero=None, bias=None):
    """(result, sum of the magnitudes of its terms)."""
    group = x.shape[1] // scale.shape[1]
    full = weights(w, zero, group) * scale.double().repeat_interleave(group, 1)
    out, size = x.double() @ full.t(), x.double().abs() @ full.abs().t()
    if bias is not None:
        out, size = out + bias.double(), size + bias.double().abs()
    return out, size


def quantise(y, dtype):
    """Nearest code, ties to even, saturating; NaN stays NaN and is 0 as an integer."""
    y = torch.clamp(y, -QMAX[dtype], QMAX[dtype])
    if dtype == S8:
        return torch.round(torch.nan_to_num(y)).to(S8)
    bits, least = {E4M3: (3, -6), E5M2: (2, -14)}[dtype]
    exponent = torch.clamp(torch.frexp(y)[1] - 1, min=least) - bits
    return torch.ldexp(torch.round(torch.ldexp(y, -exponent)), exponent).to(torch.float32).to(dtype)


def append(k_new, v_new, k_pages, v_pages, k_scale, v_scale, table, lens, new_lens=None):
    """The cache after the call; the arguments are left as they are."""
    result = []
    for new, pages, scales in ((k_new, k_pages, k_scale), (v_new, v_pages, v_scale)):
        raw, scales, dtype = pages.clone().view(torch.uint8), scales.clone(), pages.dtype
        page = pages.shape[2]
        for b, length in enumerate(lens.tolist()):
            count = new.shape[1] if new_lens is None else min(max(int(new_lens[b]), 0), new.shape[1])
            begin = length - count
            for j in range(max(begin, 0) // page, -(-length // page)):
                first, last = max(begin, j * page, 0), min(length, (j + 1) * page)
                at = int(table[b, j]) if j < table.shape[1] else -1
                if first >= last or not 0 <= at < pages.shape[0]:
                    continue
                for h in range(pages.shape[1]):
                    x = new[b, first - begin:last - begin, h].double()
                    top = torch.where(torch.isfinite(x), x.abs(), 0.0).max()
                    fraction, power = torch.frexp(top / QMAX[dtype])
                    scale = 2.0 ** max(int(power) - (1 if float(fraction) == 0.5 else 0), -126) if top > 0 else 2.0 ** -126
                    held = first - j * page
                    if held:
                        scale = max(scale, float(scales[at, h]))
                        old = raw[at, h, :held].view(dtype).double() * float(scales[at, h])
                        raw[at, h, :held] = quantise((old.float() / torch.tensor(scale, device=old.device)).double(), dtype).view(torch.uint8)
                    raw[at, h, held:held + last - first] = quantise((x.float() / torch.tensor(scale, device=x.device)).double(), dtype).view(torch.uint8)
                    scales[at, h] = scale
        result += [raw.view(dtype), scales]
    return result[0], result[2], result[1], result[3]


def attention(q, k_pages, v_pages, k_scale, v_scale, table, lens, new_lens=None, softmax_scale=None, window=0):
    """(out, lse, sum of p |v|, bound on the error of a score in f32 products), all in 64 bits."""
    batch, new, heads, dim = q.shape
    kv_heads, page = k_pages.shape[1:3]
    c = dim ** -0.5 if softmax_scale is None else softmax_scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, slack = torch.zeros_like(out), torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lens.tolist()):
        count = new if new_lens is None else min(max(int(new_lens[b]), 0), new)
        used = table[b, :max(0, min(-(-length // page), table.shape[1]))].long()
        good = ((used >= 0) & (used < k_pages.shape[0])).repeat_interleave(page)
        used = used.clamp(0, k_pages.shape[0] - 1)
        for h in range(heads):
            kv = h // (heads // kv_heads)
            k, v = ((take(p, (used, kv)).double() * s[used, kv].double()[:, None, None]).reshape(-1, dim) for p, s in ((k_pages, k_scale), (v_pages, v_scale)))
            for i in range(count):
                end = length - count + i + 1
                begin = max(0, end - window) if window else 0
                at = torch.arange(begin, max(begin, min(end, k.shape[0])), device=q.device)
                at = at[good[at]]
                if not len(at):
                    continue
                x = q[b, i, h].double()
                s = (k[at] @ x) * c
                lse[b, i, h] = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                out[b, i, h], size[b, i, h] = p @ v[at], p @ v[at].abs()
                slack[b, i, h] = dim * 2.0 ** -23 * abs(c) * (k[at].abs() @ x.abs()).max() + len(at) * 2.0 ** -24
    return out, lse, size, slack


def make_cache(pages, kv_heads, page, dim, dtype, device, seed=0):
    """Codes over the type's range and scales that make the values about 1."""
    g = torch.Generator().manual_seed(seed)
    shape = (pages, kv_heads, page, dim)

    def codes():
        if dtype == S8:
            return torch.randint(-127, 128, shape, generator=g).to(S8).to(device)
        return torch.clamp(torch.randn(shape, generator=g) * QMAX[dtype] / 6, -QMAX[dtype], QMAX[dtype]).to(dtype).to(device)

    k, v = codes(), codes()
    scales = ((torch.rand((2, pages, kv_heads), generator=g) * 1.5 + 0.5) * 3 / QMAX[dtype]).to(device)
    return k, v, scales[0].contiguous(), scales[1].contiguous()


def make_table(lens, page, pages, device, seed=0, behind=-1, width=None):
    """Each sequence's pages at random places, `behind` after its last."""
    counts = [max(0, -(-n // page)) for n in lens]
    width = max([1] + counts) if width is None else width
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
    table = torch.full((len(lens), width), behind, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :min(n, width)] = order[at:at + n][:width]
        at += n
    assert at <= pages
    return table.to(device)
