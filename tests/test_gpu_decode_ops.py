"""The decode-step operators on the device against their 64-bit forms, where they can go wrong."""
import math

import pytest
import torch

import decode_reference as ref
import xla_b200
from decode_reference import E4M3, E5M2, HALF_STEP, S8

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _status():
    torch.cuda.synchronize()
    return xla_b200.device_status()


# ---- the dot with 4-bit weights ---------------------------------------------------------------
def _dot_inputs(dev, m, n, k, group, dtype, zeros, bias, scale_dtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g).to(dtype)
    w = torch.randint(0, 256, (n, k // 2), generator=g).to(torch.uint8)
    scale = (torch.rand((n, k // group), generator=g) + 0.5).to(scale_dtype or dtype)
    zero = torch.randint(0, 16, (n, k // group), generator=g).to(torch.uint8) if zeros else None
    b = torch.randn((n,), generator=g).to(dtype) if bias else None
    return [None if t is None else t.to(dev) for t in (x, w, scale, zero, b)]


def _check_dot(out, inputs, k):
    want, size = ref.dot(*inputs)
    # Products of integers below 32 and 11-bit values are exact in f32; each of the k + groups + 1 additions and the
    # multiplications by the scales is off by at most one step of 2^-23 of the magnitudes summed; D is rounded once.
    tolerance = (k + 2 * inputs[2].shape[1] + 2) * 2.0 ** -23 * size + HALF_STEP[out.dtype] * (1 + 2.0 ** -10) * want.abs()
    off = (out.double() - want).abs()
    assert bool((off <= tolerance).all()), float((off - tolerance).max())
    # The additions' errors are independent of one another, about sqrt(k) steps of the result and not k of the terms.
    norm = float(want.norm())
    assert float(off.norm()) <= (HALF_STEP[out.dtype] + 4 * math.sqrt(k) * 2.0 ** -23) * norm + 1e-30


@pytest.mark.parametrize("m,n,k,group,dtype,zeros,bias", [
    (1, 256, 512, 128, BF16, False, False),
    (1, 1, 32, 32, F16, False, True),
    (1, 17, 64, 64, BF16, True, False),
    (1, 130, 4096, 64, F16, True, True),
    (2, 33, 160, 32, BF16, False, True),
    (3, 1000, 1024, 128, F16, False, False),
    (5, 515, 4416, 32, F16, True, True),
    (7, 15, 8192, 128, BF16, True, False),
    (8, 2048, 2048, 64, BF16, False, False),
    (9, 16, 96, 32, F16, False, True),
    (16, 300, 1152, 128, BF16, True, True),
    (17, 129, 640, 64, BF16, True, False),
    (31, 77, 256, 256, F16, False, False),
    (32, 512, 3200, 128, BF16, False, True),
    (33, 31, 1920, 64, F16, True, False),
    (64, 200, 1536, 512, BF16, True, True),
    (64, 5, 64, 32, F16, False, False),
])
def test_dot_w4(cuda_device, m, n, k, group, dtype, zeros, bias):
    inputs = _dot_inputs(cuda_device, m, n, k, group, dtype, zeros, bias, seed=m * n + k)
    x, w, scale, zero, b = inputs
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, bias=b), inputs, k)
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, bias=b, out_dtype=F32), inputs, k)
    assert _status() == 0


@pytest.mark.parametrize("m,n,k,group,dtype,zeros,bias", [
    (1, 19000, 4096, 128, F16, False, False),      # one or two rows of x against many rows of weights: x is converted first
    (1, 40000, 4096, 256, BF16, True, True),       # more blocks of rows than the sums have room for
    (1, 4800, 4224, 32, BF16, False, True),
    (1, 19000, 4160, 64, F16, True, False),        # k ends inside a step
    (2, 28500, 4096, 128, BF16, False, True),
    (2, 9600, 4128, 32, F16, True, True),
    (2, 28500, 12288, 384, BF16, True, False),
    (1, 4800, 32768, 32, F16, False, False),       # ... which does not fit any more
    (20, 80000, 160, 32, BF16, True, True),        # more rows than a CTA's warps take at once
    (32, 76300, 2080, 32, F16, False, True),       # ... and x in several phases, k ending inside a step
    (3, 75777, 96, 32, BF16, False, False),
    (12, 1000, 5152, 32, BF16, True, False),
    (9, 150, 28672, 128, F16, True, True),
    (32, 2500, 11008, 64, BF16, False, True),
    (47, 2400, 4160, 64, BF16, False, True),
])
def test_dot_w4_large(cuda_device, m, n, k, group, dtype, zeros, bias):
    inputs = _dot_inputs(cuda_device, m, n, k, group, dtype, zeros, bias, seed=m + n + k)
    x, w, scale, zero, b = inputs
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, bias=b), inputs, k)
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, bias=b, out_dtype=F32), inputs, k)
    assert _status() == 0


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 32, 33, 48, 49, 100, 177, 250, 481, 511, 512])
def test_dot_w4_rows_of_a_cta(cuda_device, rows):
    """Every split of a CTA's warps: this many rows of weights each, and one more for some of them."""
    for m, group, dtype, zeros in ((5, 64, F16, True), (20, 128, BF16, False)):
        inputs = _dot_inputs(cuda_device, m, 148 * rows + 3, 1280, group, dtype, zeros, True)
        _check_dot(xla_b200.dot_w4(*inputs[:3], zero=inputs[3], bias=inputs[4]), inputs, 1280)
    assert _status() == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("scale_dtype", [F32, F16, BF16])
def test_dot_w4_scale_types_of_many_rows(cuda_device, scale_dtype, group):
    for dtype, zeros in ((BF16, False), (F16, True)):
        inputs = _dot_inputs(cuda_device, 1, 19000, 4096, group, dtype, zeros, False, scale_dtype)
        _check_dot(xla_b200.dot_w4(*inputs[:3], zero=inputs[3]), inputs, 4096)


def test_dot_w4_many_rows_large_magnitudes_and_infinities(cuda_device):
    x, w, scale, _, _ = _dot_inputs(cuda_device, 2, 9600, 4096, 32, BF16, False, False)
    x[0] *= 2.0 ** 100
    x[1] *= 2.0 ** -100
    _check_dot(xla_b200.dot_w4(x, w, scale, out_dtype=F32), [x, w, scale, None, None], 4096)
    for value in (math.inf, -math.inf, math.nan):
        x[1, 17] = value
        out = xla_b200.dot_w4(x, w, scale, out_dtype=F32)
        _check_dot(out[:1], [x[:1], w, scale, None, None], 4096)
        want = value * ref.weights(w, None, 32)[:, 17]
        assert torch.equal(out[1].isposinf(), want.isposinf()) and torch.equal(out[1].isneginf(), want.isneginf()) and torch.equal(out[1].isnan(), want.isnan())


@pytest.mark.parametrize("m,n,k,group,dtype,zeros,bias,scale_dtype", [
    (1, 1, 32, 32, BF16, False, True, F32),        # groups of 32: any size ...
    (1, 7, 64, 32, F16, True, False, BF16),
    (1, 300, 96, 32, BF16, True, True, F16),
    (1, 5003, 4416, 32, F16, False, True, F16),
    (2, 100, 2080, 32, F16, True, False, F32),
    (2, 9, 8192, 32, BF16, False, True, BF16),
    (2, 300, 1024, 32, BF16, True, True, BF16),    # ... but not a short k for two rows
    (1, 77, 32768, 32, F16, True, True, F32),      # and x has to fit
    (1, 50000, 4096, 128, F16, True, True, F32),   # longer groups: 200 million weights
    (1, 50001, 4096, 256, BF16, True, False, BF16),
    (1, 49000, 4160, 64, F16, False, True, F16),   # k ends inside a step
    (1, 49000, 4160, 64, BF16, True, True, F32),
    (2, 49000, 4224, 384, BF16, False, True, BF16),
    (2, 49000, 4160, 64, F16, False, False, F32),
    (1, 20000, 12800, 640, F16, True, True, BF16),
    (2, 50000, 4096, 128, F16, True, True, F16),   # not two rows with zero points
])
def test_dot_w4_of_one_and_two_rows(cuda_device, m, n, k, group, dtype, zeros, bias, scale_dtype):
    """Both sides of the choice between the two kernels."""
    inputs = _dot_inputs(cuda_device, m, n, k, group, dtype, zeros, bias, scale_dtype, seed=m + n + k)
    x, w, scale, zero, b = inputs
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, bias=b), inputs, k)
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, bias=b, out_dtype=F32), inputs, k)
    x[m - 1, k - 1] = math.inf                     # reaches its own row only, with the sign of the last weight
    out = xla_b200.dot_w4(x, w, scale, zero=zero, out_dtype=F32)
    if m == 2:
        _check_dot(out[:1], [x[:1], w, scale, zero, None], k)
    last = ref.weights(w[:, -1:], None if zero is None else zero[:, -1:], 2)[:, 1]
    assert torch.equal(out[m - 1].isposinf(), last > 0) and torch.equal(out[m - 1].isneginf(), last < 0) and torch.equal(out[m - 1].isnan(), last == 0)
    assert _status() == 0


def test_dot_w4_every_nibble_of_many_rows_and_longer_groups(cuda_device):
    """Powers of two at one place of k: exact, for every nibble and zero point, in groups of 64 and 128."""
    n, k = 50000, 4096
    w = (torch.arange(n * k // 2, device=cuda_device) * 2654435761 // 65536 % 256).to(torch.uint8).reshape(n, k // 2)
    for group in (64, 128):
        scale = torch.ones((n, k // group), dtype=F32, device=cuda_device)
        for zero in (None, (torch.arange(n * k // group, device=cuda_device) % 16).to(torch.uint8).reshape(n, k // group)):
            for at in (0, 3, 6, 31, 32, 77, 127, 2050, 4095):
                x = torch.zeros((1, k), dtype=BF16, device=cuda_device)
                x[0, at] = -2.0 ** (at % 7)
                byte = w[:, at // 2] >> (4 * (at % 2)) & 15
                want = (byte ^ 8).double() - 8 if zero is None else byte.double() - zero[:, at // group].double()
                assert torch.equal(xla_b200.dot_w4(x, w, scale, zero=zero, out_dtype=F32)[0].double(), want * -2.0 ** (at % 7))


@pytest.mark.parametrize("m,n,k,group,dtype,zeros,outlier", [
    (1, 50000, 4096, 128, BF16, False, 99840.0),
    (1, 50000, 4096, 128, F16, True, 60000.0),
    (1, 50000, 4096, 64, BF16, True, 2.0 ** 24),
    (1, 9600, 4096, 32, F16, False, 60000.0),
    (2, 60000, 4096, 128, BF16, False, 99840.0),
    (2, 20000, 4096, 32, BF16, True, 2.0 ** 24),
    (3, 2000, 4096, 128, BF16, True, 99840.0),
])
def test_dot_w4_outliers_of_x_where_the_weight_is_its_zero_point(cuda_device, m, n, k, group, dtype, zeros, outlier):
    """Such a value of x adds nothing, and must not cost the other terms any bits: w - z is formed before the products.

    The bounds of _check_dot hold as they stand, for the terms at the outliers are zeros in them.  Beside an outlier of 2^24 a
    value of x may be off by 2^-40 of it, 2^-16, if it lies more than 2^32 below it, as three in a thousand normal values
    do: that moves the results by less than sqrt(0.0032) 2^-16 = 9e-7 of their size, a thirtieth of the bound."""
    x, w, scale, zero, _ = inputs = _dot_inputs(cuda_device, m, n, k, group, dtype, zeros, False, seed=n + group)
    for row in range(m):
        for at in (5 + 2 * row, 777 + row, k - 2 - row):
            x[row, at] = outlier * (-1) ** at
            z = zero[:, at // group] if zeros else torch.zeros(n, dtype=torch.uint8, device=cuda_device)
            byte = w[:, at // 2]
            w[:, at // 2] = (byte & 0xF0) | z if at % 2 == 0 else (byte & 0x0F) | (z << 4)
    assert torch.equal(ref.weights(w, zero, group)[:, 777], torch.zeros(n, dtype=torch.float64, device=cuda_device))
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero, out_dtype=F32), inputs, k)
    _check_dot(xla_b200.dot_w4(x, w, scale, zero=zero), inputs, k)
    assert _status() == 0


@pytest.mark.parametrize("n,k,group,dtype,zeros", [
    (5488, 608, 32, F16, False),
    (1000, 2048, 32, F16, True),
    (5488, 608, 32, BF16, True),
    (50000, 4096, 128, F16, True),
    (50000, 4096, 64, BF16, False),
])
@pytest.mark.parametrize("m", [1, 3])
def test_dot_w4_sums_keep_the_bits_of_f32(cuda_device, m, n, k, group, dtype, zeros):
    """One large value of x and its products, of at most 11 + 5 bits, in the same sums as all the others.

    At most 64 additions follow one another: a warp's products (8 for 128 of k, every 16th or 24th step), its groups, and the
    sums of up to 24 warps; each is off by at most a step of 2^-23 of a sum that is no larger than about the result."""
    x, w, scale, zero, _ = inputs = _dot_inputs(cuda_device, m, n, k, group, dtype, zeros, False, F32, seed=n + k)
    x[:, k // 3] = 7720.0
    out = xla_b200.dot_w4(x, w, scale, zero=zero, out_dtype=F32)
    want, _ = ref.dot(*inputs)
    assert float((out.double() - want).norm() / want.norm()) <= 8 * 2.0 ** -23


def test_dot_w4_many_rows_one_value_at_a_time(cuda_device):
    """Powers of two at one place of k: exact, for every nibble and zero point."""
    n, k = 4800, 4096
    w = (torch.arange(n * k // 2, device=cuda_device) * 2654435761 // 65536 % 256).to(torch.uint8).reshape(n, k // 2)
    scale = torch.ones((n, k // 32), dtype=F32, device=cuda_device)
    for zero in (None, (torch.arange(n * k // 32, device=cuda_device) % 16).to(torch.uint8).reshape(n, k // 32)):
        full = ref.weights(w, zero, 32)
        for at in (0, 1, 2, 3, 4, 5, 6, 7, 45, 127, 128, 2047, 4095):
            x = torch.zeros((1, k), dtype=F16, device=cuda_device)
            x[0, at] = 2.0 ** (at % 5)
            assert torch.equal(xla_b200.dot_w4(x, w, scale, zero=zero, out_dtype=F32)[0].double(), full[:, at] * 2.0 ** (at % 5))


@pytest.mark.parametrize("scale_dtype", [F32, F16, BF16])
def test_dot_w4_scale_types(cuda_device, scale_dtype):
    for dtype in (BF16, F16):
        inputs = _dot_inputs(cuda_device, 4, 96, 768, 64, dtype, True, False, scale_dtype)
        _check_dot(xla_b200.dot_w4(inputs[0], inputs[1], inputs[2], zero=inputs[3]), inputs, 768)


def test_dot_w4_every_nibble_and_zero_point(cuda_device):
    """One group whose weights are all 256 bytes' nibbles, against x of one 1 at a time: exact."""
    k = 512
    w = torch.arange(256, dtype=torch.uint8).reshape(1, 256).expand(16, 256).contiguous().to(cuda_device)
    x = torch.zeros((32, k), dtype=F16, device=cuda_device)
    for zero in (None, torch.arange(16, dtype=torch.uint8, device=cuda_device).reshape(16, 1).expand(16, 4).contiguous()):
        scale = torch.ones((16, 4), dtype=F32, device=cuda_device)
        for start in range(0, k, 32):
            x.zero_()
            x[torch.arange(32), start + torch.arange(32)] = 1
            got = xla_b200.dot_w4(x, w, scale, zero=zero, out_dtype=F32)
            assert torch.equal(got.double(), ref.dot(x, w, scale, zero)[0])


def test_dot_w4_large_magnitudes_and_infinities(cuda_device):
    x, w, scale, _, _ = _dot_inputs(cuda_device, 3, 40, 256, 64, BF16, False, False)
    x[0] *= 2.0 ** 100
    x[1] *= 2.0 ** -100
    x[2, 17] = math.inf
    out = xla_b200.dot_w4(x, w, scale, out_dtype=F32)
    _check_dot(out[:2], [x[:2], w, scale, None, None], 256)
    full = ref.weights(w, None, 64)[:, 17]
    assert torch.equal(out[2].isposinf(), full > 0) and torch.equal(out[2].isneginf(), full < 0) and torch.equal(out[2].isnan(), full == 0)


def test_dot_w4_no_rows_and_neighbours_untouched(cuda_device):
    x, w, scale, _, _ = _dot_inputs(cuda_device, 5, 37, 128, 32, F16, False, False)
    assert xla_b200.dot_w4(x[:0], w, scale).shape == (0, 37)
    big = torch.full((9, 37), 7.0, dtype=F16, device=cuda_device)
    xla_b200.dot_w4(x, w, scale, out=big[2:7])
    assert bool((big[:2] == 7).all()) and bool((big[7:] == 7).all())
    _check_dot(big[2:7], [x, w, scale, None, None], 128)


def test_dot_w4_same_result_every_time(cuda_device):
    x, w, scale, zero, b = _dot_inputs(cuda_device, 6, 1000, 4096, 128, BF16, True, True)
    first = xla_b200.dot_w4(x, w, scale, zero=zero, bias=b, out_dtype=F32)
    assert all(torch.equal(first, xla_b200.dot_w4(x, w, scale, zero=zero, bias=b, out_dtype=F32)) for _ in range(5))


# ---- appending to the cache --------------------------------------------------------------------
def _append_inputs(dev, batch, new, kv_heads, dim, page, lens, code, dtype, new_lens=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    pages = sum(max(0, -(-n // page)) for n in lens) + 2
    k, v, ks, vs = ref.make_cache(pages, kv_heads, page, dim, code, dev, seed)
    ks, vs = torch.exp2(torch.round(torch.log2(ks))), torch.exp2(torch.round(torch.log2(vs)))
    fresh = [(torch.randn((batch, new, kv_heads, dim), generator=g) * torch.exp2(torch.randint(-6, 5, (batch, new, kv_heads, 1), generator=g))).to(dtype).to(dev) for _ in range(2)]
    table = ref.make_table(lens, page, pages, dev, seed)
    lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    new_lens = None if new_lens is None else torch.tensor(new_lens, dtype=torch.int32, device=dev)
    return fresh + [k, v, ks, vs, table, lens], new_lens


def _check_append(args, new_lens):
    want = ref.append(*args, new_lens)
    xla_b200.kv_cache_append(*args, new_lens=new_lens)
    for got, expected in zip(args[2:6], want):
        assert torch.equal(got.view(torch.uint8), expected.view(torch.uint8))


@pytest.mark.parametrize("batch,new,kv_heads,dim,page,lens,code,dtype,new_lens", [
    (1, 1, 1, 16, 16, [1], E4M3, BF16, None),
    (3, 1, 2, 64, 16, [16, 17, 33], S8, F16, None),
    (4, 1, 8, 128, 64, [1, 64, 65, 200], E4M3, BF16, None),
    (2, 5, 3, 80, 32, [5, 70], E5M2, BF16, None),
    (2, 33, 2, 96, 16, [40, 49], E4M3, F16, [33, 7]),
    (3, 100, 1, 256, 128, [100, 128, 300], S8, BF16, [100, 0, 99]),
    (2, 64, 2, 128, 64, [64, 129], E5M2, F16, [64, 64]),
    (2, 3, 2, 48, 16, [2, 0], E4M3, BF16, [2, 0]),
])
def test_append(cuda_device, batch, new, kv_heads, dim, page, lens, code, dtype, new_lens):
    args, fresh = _append_inputs(cuda_device, batch, new, kv_heads, dim, page, lens, code, dtype, new_lens, seed=sum(lens))
    _check_append(args, fresh)
    _check_append(args, fresh)          # again at the same place: the same cache
    assert _status() == 0


@pytest.mark.parametrize("batch,new,kv_heads,dim,page,lens,code,dtype,new_lens", [
    (1, 300, 1, 256, 128, [310], E4M3, BF16, None),           # a lane has more pieces than it keeps
    (2, 130, 2, 16, 16, [133, 140], E5M2, F16, [130, 9]),     # nine pages of one call, several to a block
    (3, 70, 2, 64, 32, [70, 100, 69], S8, BF16, [70, 70, 69]),
    (100, 1, 1, 32, 16, list(range(100)), E4M3, F16, [min(i, 1) for i in range(100)]),
])
def test_append_many_pages(cuda_device, batch, new, kv_heads, dim, page, lens, code, dtype, new_lens):
    args, fresh = _append_inputs(cuda_device, batch, new, kv_heads, dim, page, lens, code, dtype, new_lens, seed=sum(lens))
    _check_append(args, fresh)
    args[0][0, 0, 0, 3], args[1][0, -1, 0, 5], args[0][-1, -1, -1, -1] = math.inf, -math.inf, math.nan
    _check_append(args, fresh)
    assert _status() == 0


@pytest.mark.parametrize("code", [E4M3, E5M2, S8])
def test_append_token_by_token_grows_the_scale(cuda_device, code):
    """Tokens of growing size, one call each: every step equals the definition's."""
    page, dim = 16, 32
    k, v, ks, vs = ref.make_cache(3, 1, page, dim, code, cuda_device)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=cuda_device)
    g = torch.Generator().manual_seed(3)
    for t in range(20):
        k_new, v_new = ((torch.randn((1, 1, 1, dim), generator=g) * 2.0 ** (t / 2 - 4)).to(BF16).to(cuda_device) for _ in range(2))
        _check_append([k_new, v_new, k, v, ks, vs, table, torch.tensor([t + 1], dtype=torch.int32, device=cuda_device)], None)


@pytest.mark.parametrize("code", [E4M3, E5M2, S8])
@pytest.mark.parametrize("value", [0.0, ref.QMAX[E4M3], 449.0, 127.0, 128.0, 57344.0, 1e-40, 3e38, math.inf, -math.inf, math.nan])
def test_append_values_at_the_borders(cuda_device, code, value):
    k_new = torch.full((1, 2, 1, 16), 0.75, dtype=BF16, device=cuda_device)
    k_new[0, 0, 0, 3] = value
    v_new = torch.full_like(k_new, value)
    k, v, ks, vs = ref.make_cache(2, 1, 16, 16, code, cuda_device)
    args = [k_new, v_new, k, v, ks, vs, torch.tensor([[1]], dtype=torch.int32, device=cuda_device), torch.tensor([2], dtype=torch.int32, device=cuda_device)]
    _check_append(args, None)


def test_append_to_pages_with_other_scales(cuda_device):
    """Scales that are no powers of two, as another quantiser leaves them."""
    args, _ = _append_inputs(cuda_device, 3, 2, 2, 64, 16, [9, 20, 34], E4M3, BF16)
    args[4].mul_(1.3)
    args[5].mul_(0.7)
    _check_append(args, None)


def test_append_with_padding_in_front(cuda_device):
    """Sequences shorter than their new tokens: the first of them are padding."""
    args, _ = _append_inputs(cuda_device, 4, 20, 2, 32, 16, [0, 1, 17, 20], E4M3, BF16)
    _check_append(args, None)
    assert _status() == 0


def test_append_reports_pages_outside_of_the_cache(cuda_device):
    args, _ = _append_inputs(cuda_device, 2, 2, 1, 32, 16, [17, 20], E4M3, BF16)
    args[6][0, 1] = 10 ** 6                    # the second token of sequence 0 has no page
    args[7][1] = 100                           # sequence 1 is longer than its table
    _check_append(args, None)
    assert _status() == 64 and _status() == 0


# ---- attention ---------------------------------------------------------------------------------
def _attention_inputs(dev, heads, kv_heads, dim, page, lens, new, code, dtype, seed=0, sharp=2.0):
    pages = sum(max(0, -(-n // page)) for n in lens) + 2
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((len(lens), new, heads, dim), generator=g) * sharp).to(dtype).to(dev)
    cache = ref.make_cache(pages, kv_heads, page, dim, code, dev, seed)
    return [q, *cache, ref.make_table(lens, page, pages, dev, seed), torch.tensor(lens, dtype=torch.int32, device=dev)]


def _attention_tolerance(want, size, slack, dtype):
    # A weight is off by its rounding to 11 bits (relative 2^-11), by the error of its score (slack, twice: it is in the
    # weight and in the sum) and by a few steps of exp2 and of the rescalings; the output is rounded once.
    return size * (2.0 ** -11 * (1 + 2.0 ** -6) + 2 * slack[..., None] + 2.0 ** -18) + HALF_STEP[dtype] * (1 + 2.0 ** -7) * want.abs() + 2.0 ** -25


def _check_attention(args, new_lens=None, window=0, scale=None, out=None):
    new_lens = None if new_lens is None else torch.tensor(new_lens, dtype=torch.int32, device=args[0].device)
    got, lse = out if out is not None else xla_b200.paged_attention_kv8(*args, new_lens=new_lens, window=window, softmax_scale=scale, return_lse=True)
    want, want_lse, size, slack = ref.attention(*args, new_lens, scale, window)
    tolerance = _attention_tolerance(want, size, slack, got.dtype)
    off = (got.double() - want).abs()
    assert bool((off <= tolerance).all()), float((off - tolerance).max())
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and bool((got[empty] == 0).all())
    close = (lse.double() - want_lse)[~empty].abs() <= (slack + 2.0 ** -18 + want_lse.abs() * 2.0 ** -22)[~empty]
    assert bool(close.all())


@pytest.mark.parametrize("heads,kv_heads,dim,page,lens,new,code,dtype,new_lens,window", [
    (1, 1, 16, 16, [1], 1, E4M3, BF16, None, 0),
    (8, 2, 64, 16, [37], 1, E4M3, F16, None, 0),
    (8, 1, 128, 16, [0, 1, 15, 16, 17, 63, 64, 65], 1, E4M3, BF16, None, 0),
    (32, 8, 128, 64, [300, 5, 64], 1, E4M3, BF16, None, 0),
    (4, 4, 80, 32, [129, 31], 1, E5M2, BF16, None, 0),
    (5, 1, 96, 16, [100], 1, S8, F16, None, 0),
    (16, 1, 112, 16, [77, 200], 1, E5M2, F16, None, 0),
    (6, 2, 256, 16, [130, 47], 1, E4M3, F16, None, 0),
    (40, 1, 192, 64, [190], 1, S8, BF16, None, 0),
    (16, 4, 128, 32, [5, 40, 130], 5, S8, BF16, None, 0),
    (8, 2, 64, 16, [8, 3, 100], 8, E4M3, F16, [8, 3, 2], 0),
    (64, 8, 128, 128, [1000, 129], 3, E4M3, BF16, [0, 3], 0),
    (8, 2, 128, 16, [500, 20, 1], 1, E4M3, BF16, None, 33),
    (8, 2, 64, 64, [300, 65], 7, E5M2, BF16, None, 1),
    (4, 2, 128, 32, [200], 64, E4M3, BF16, None, 100),
    (2, 1, 32, 16, [64], 64, S8, F16, None, 0),
    (8, 8, 256, 128, [700], 2, E5M2, BF16, None, 0),
    (256, 1, 64, 16, [90, 1], 1, E4M3, BF16, None, 0),
    (60, 4, 128, 64, [700, 130], 3, S8, F16, [3, 1], 0),
    (1, 1, 16, 16, [i % 23 for i in range(1500)], 1, E5M2, F16, [min(i % 23, 1) for i in range(1500)], 0),
    (2, 1, 48, 16, [2000 - i for i in range(40)], 2, S8, BF16, None, 0),
])
def test_attention(cuda_device, heads, kv_heads, dim, page, lens, new, code, dtype, new_lens, window):
    args = _attention_inputs(cuda_device, heads, kv_heads, dim, page, lens, new, code, dtype, seed=sum(lens) + dim)
    _check_attention(args, new_lens, window)
    assert _status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,page,lens,new,code", [
    (8, 2, 64, 16, [37, 500], 1, E4M3),
    (6, 1, 256, 16, [1000, 47], 1, E4M3),
    (16, 1, 128, 32, [300, 90], 3, S8),
    (5, 1, 96, 64, [9000], 1, E5M2),
    (32, 2, 64, 128, [2000, 77], 1, S8),
    (40, 4, 128, 32, [5000, 5], 5, S8),
])
def test_attention_of_f16_is_rounded_once(cuda_device, heads, kv_heads, dim, page, lens, new, code):
    """The weights of f16 results are no coarser than the sums: only the last rounding is one to 11 bits.

    The bound is _attention_tolerance's without the weights' 2^-11: each weight is held to 2^-22, below its 2^-18."""
    args = _attention_inputs(cuda_device, heads, kv_heads, dim, page, lens, new, code, F16, seed=dim)
    want, _, size, slack = ref.attention(*args)
    off = (xla_b200.paged_attention_kv8(*args).double() - want).abs()
    tolerance = size * (2 * slack[..., None] + 2.0 ** -18) + HALF_STEP[F16] * (1 + 2.0 ** -7) * want.abs() + 2.0 ** -25
    assert bool((off <= tolerance).all()), float((off / tolerance).max())
    nearest = want.to(F16).double() - want                   # what the last rounding alone leaves
    assert float(off.norm()) <= 1.01 * float(nearest.norm())


def test_attention_of_long_and_short_sequences_together(cuda_device):
    """One sequence far longer than the others: its work is split over the card and joined."""
    for dtype, new in ((BF16, 1), (F16, 2)):
        args = _attention_inputs(cuda_device, 4, 1, 128, 64, [3, 20000, 64, 0, 7001], new, E4M3, dtype)
        _check_attention(args, [min(n, new) for n in (3, 20000, 64, 0, 7001)])
    _check_attention(_attention_inputs(cuda_device, 6, 3, 64, 16, [9000], 1, S8, BF16), window=5000)
    for window in (300, 351, 352, 600):
        _check_attention(_attention_inputs(cuda_device, 8, 2, 128, 64, [5000, 40, 700], 17, E4M3, BF16), window=window)
    _check_attention(_attention_inputs(cuda_device, 2, 1, 256, 128, [6000, 1], 1, E4M3, BF16))


@pytest.mark.parametrize("lens,kv_heads", [([131072] + [0] * 15, 1), ([5, 0, 131072, 40], 1), ([131072], 1), ([0] * 63 + [100000], 2), ([131072, 131072], 1)])
def test_attention_cuts_a_sequence_into_a_limited_number_of_pieces(cuda_device, lens, kv_heads):
    """Idle and short sequences beside a long one do not add to its pieces, which one warp joins for each row.

    Each CTA leaves word of the item that the end of its share cuts, (sequence, item, pieces, new tokens), at the workspace's
    end.  A share is no smaller than the largest item over 128, to the nearest unit and two at least: 320 units in shares of
    two and a half, or 319 in shares of two, are 160 pieces at most, and the item's ends may lie inside of shares."""
    args = _attention_inputs(cuda_device, 4 * kv_heads, kv_heads, 128, 64, lens, 1, E4M3, BF16)
    fresh = torch.tensor([min(n, 1) for n in lens], dtype=torch.int32, device=cuda_device)
    work = torch.zeros(xla_b200.paged_attention_workspace_bytes(len(lens), 1, 4 * kv_heads, kv_heads, 128), dtype=torch.int8, device=cuda_device)
    out = xla_b200.paged_attention_kv8(*args, new_lens=fresh, workspace=work, return_lse=True)
    pieces = work[-148 * 5 * 16:].view(torch.int32).reshape(-1, 4)[:, 2]
    assert 64 <= int(pieces.max()) <= 162, int(pieces.max())
    _check_attention(args, fresh.tolist(), out=out)


def test_attention_of_many_sequences(cuda_device):
    """More sequences than a warp has lanes, their work in shares that begin and end anywhere."""
    for heads, kv_heads, dim, new, code in ((8, 2, 64, 1, E4M3), (16, 1, 128, 2, S8), (2, 2, 256, 1, E5M2)):
        g = torch.Generator().manual_seed(dim)
        lens = (torch.randint(0, 900, (70,), generator=g) * (torch.rand(70, generator=g) < 0.8)).tolist()
        lens[33] = 3000
        args = _attention_inputs(cuda_device, heads, kv_heads, dim, 32, lens, new, code, BF16)
        _check_attention(args, [min(n, new) for n in lens])
        _check_attention(args, [min(n, new) for n in lens], window=200)
    assert _status() == 0


@pytest.mark.parametrize("window", [2 ** 30 - 1, 2 ** 30, 2 ** 31, 2 ** 63 - 64, 2 ** 63 - 1])
def test_attention_with_a_window_larger_than_any_sequence(cuda_device, window):
    """Such a window is none, and the work is split over the card as without one: the second launch joins it."""
    args = _attention_inputs(cuda_device, 4, 1, 128, 64, [9000, 70], 2, E4M3, BF16)
    want = xla_b200.paged_attention_kv8(*args, return_lse=True)
    before = xla_b200.launch_count()
    got = xla_b200.paged_attention_kv8(*args, window=window, return_lse=True)
    assert xla_b200.launch_count() - before == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _check_attention(args, window=window, out=got)


def test_attention_keeps_a_bad_page_scale_to_the_rows_that_see_it(cuda_device):
    """The second drafted token opens a page whose scales are no numbers: the first token's rows do not see it."""
    for bad in (math.nan, math.inf):
        args = _attention_inputs(cuda_device, 4, 2, 128, 16, [33], 2, E4M3, BF16)
        want, want_lse, size, slack = ref.attention(*args)
        for scales in args[3:5]:
            scales[int(args[5][0, 2])] = bad                 # position 32
            got, lse = xla_b200.paged_attention_kv8(*args, return_lse=True)
            assert bool(((got.double() - want).abs() <= _attention_tolerance(want, size, slack, got.dtype))[0, 0].all())
            assert bool(((lse.double() - want_lse).abs() <= slack + 2.0 ** -18 + want_lse.abs() * 2.0 ** -22)[0, 0].all())
            assert torch.equal(torch.isfinite(got[0, 1]), torch.isfinite(ref.attention(*args)[0][0, 1]))


def test_attention_scales_and_sharp_rows(cuda_device):
    """Very sharp softmax, tiny and huge queries, page scales far apart, a negative and a zero softmax scale."""
    args = _attention_inputs(cuda_device, 8, 2, 64, 16, [150, 90], 1, E4M3, BF16, sharp=8.0)
    _check_attention(args)
    _check_attention(args, scale=0.0)
    _check_attention(args, scale=-0.1)
    args[0][0, 0, 0] *= 2.0 ** -90
    args[0][0, 0, 1] *= 2.0 ** -20
    _check_attention(args)
    args[4][:] *= torch.exp2(torch.arange(args[4].shape[0], device=cuda_device) % 7 * 5.0 - 15)[:, None]
    args[4][3] = 0
    _check_attention(args)
    args[0] = args[0] * 2.0 ** 60
    args[3].mul_(2.0 ** -60)
    _check_attention(args)


@pytest.mark.parametrize("code,bits", [(E4M3, 0x7F), (E5M2, 0x7F), (E5M2, 0x7C)])
def test_attention_ignores_what_it_does_not_see(cuda_device, code, bits):
    """NaN and infinity codes behind a sequence's end, in front of a window, and in later tokens of the same call."""
    args = _attention_inputs(cuda_device, 8, 2, 128, 16, [35, 50], 3, code, BF16)
    table = args[5]
    for pages in (args[1], args[2]):
        raw = pages.view(torch.uint8)
        raw[int(table[0, 2]), :, 3:] = bits            # behind the end of sequence 0
        raw[int(table[1, 0])] = bits                   # in front of the window of sequence 1
        raw[int(table[1, 1]), :, :4] = bits
    for scales in args[3:5]:
        scales[int(table[1, 0])] = math.nan
    # A window of 30 from positions 47, 48, 49 reaches back to 18: of page 1, slots 0 and 1 are not seen ...
    for pages in (args[1], args[2]):
        pages.view(torch.uint8)[int(table[1, 1]), :, 2:4] = 0         # ... and 2, 3 are seen by some rows
    _check_attention(args, window=30)


def test_attention_keeps_a_bad_value_to_the_rows_that_see_it(cuda_device):
    """A NaN in the values of the last drafted token reaches that token's rows only."""
    for code, bits in ((E4M3, 0x7F), (E5M2, 0x7D), (E5M2, 0x7C)):
        args = _attention_inputs(cuda_device, 4, 2, 128, 16, [40], 3, code, BF16)
        want, _, size, slack = ref.attention(*args)
        args[2].view(torch.uint8)[int(args[5][0, 2]), :, 7, 5] = bits          # position 39, column 5
        got = xla_b200.paged_attention_kv8(*args)
        inside = (got.double() - want).abs() <= _attention_tolerance(want, size, slack, got.dtype)
        assert bool(inside[0, :2].all())
        assert bool((~torch.isfinite(got[0, 2, :, 5])).all())
        others = torch.arange(128, device=cuda_device) != 5
        assert bool(inside[0, 2][:, others].all())


def test_attention_reports_pages_outside_of_the_cache(cuda_device):
    args = _attention_inputs(cuda_device, 4, 2, 64, 16, [60, 33], 1, E4M3, BF16)
    args[5][0, 1] = -5
    args[5][1, 1] = 1 << 30
    _check_attention(args)
    assert _status() == 64 and _status() == 0
    args[6][0] = -7                                       # a length below 0 is an idle slot, and reported
    assert bool((xla_b200.paged_attention_kv8(*args)[0] == 0).all()) and _status() == 64
    args = _attention_inputs(cuda_device, 4, 2, 64, 16, [60, 33], 1, E4M3, BF16)
    args[6][0] = 1000                                     # a length behind the end of the table
    _check_attention(args)
    assert _status() == 64 and _status() == 0


@pytest.mark.parametrize("window", [1, 16, 100, 5000, 2 ** 30])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30 + 3, 4096 + 77, 4096 + 1])
def test_attention_of_a_length_far_outside_of_the_table(cuda_device, length, window):
    """What a window sees behind the table's end is not there, whatever the length, and the other sequences are as ever."""
    for heads, dim, new, new_lens in ((4, 128, 3, [3, 3, 3, 3]), (2, 64, 1, [1, 0, 1, 1]), (4, 256, 2, [2, 2, 0, 1])):
        args = _attention_inputs(cuda_device, heads, 2, dim, 64, [4096, 70, 4096, 0], new, E4M3, BF16)
        args[6][0] = args[6][2] = length
        _check_attention(args, new_lens, window)
        assert _status() == 64 and _status() == 0


def test_attention_over_a_cache_of_more_than_4_gib(cuda_device):
    pages, kv_heads, page, dim = 70000, 4, 128, 128        # 4.6 GB each for keys and values
    k, v = (torch.zeros((pages, kv_heads, page, dim), dtype=torch.uint8, device=cuda_device).view(E4M3) for _ in range(2))
    small = ref.make_cache(3, kv_heads, page, dim, E4M3, cuda_device)
    where = torch.tensor([69999, 33000, 66000], device=cuda_device)
    ks, vs = (torch.ones((pages, kv_heads), device=cuda_device) for _ in range(2))
    for big, part in ((k, small[0]), (v, small[1])):
        big.view(torch.uint8)[where] = part.view(torch.uint8)
    ks[where], vs[where] = small[2], small[3]
    q = torch.randn((1, 1, 8, dim), device=cuda_device).to(BF16)
    lens = torch.tensor([300], dtype=torch.int32, device=cuda_device)
    fresh = torch.randn((2, 1, 1, kv_heads, dim), device=cuda_device).to(BF16)
    table = where.to(torch.int32).reshape(1, 3)
    near = [*small, torch.arange(3, dtype=torch.int32, device=cuda_device).reshape(1, 3), lens]
    xla_b200.kv_cache_append(fresh[0], fresh[1], *near)
    xla_b200.kv_cache_append(fresh[0], fresh[1], k, v, ks, vs, table, lens)
    assert torch.equal(k.view(torch.uint8)[where], small[0].view(torch.uint8)) and torch.equal(vs[where], small[3])
    _check_attention([q, *near], out=xla_b200.paged_attention_kv8(q, k, v, ks, vs, table, lens, return_lse=True))


def test_attention_of_nothing(cuda_device):
    args = _attention_inputs(cuda_device, 4, 2, 64, 16, [0, 0], 1, E4M3, BF16)
    out, lse = xla_b200.paged_attention_kv8(*args, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all()) and _status() == 0
    none = [args[0][:0], *args[1:5], args[5][:0], args[6][:0]]
    assert xla_b200.paged_attention_kv8(*none).shape == (0, 1, 4, 64)
    assert xla_b200.paged_attention_kv8(args[0][:, :0], *args[1:]).shape == (2, 0, 4, 64)


# ---- together, on streams and in graphs ---------------------------------------------------------
def test_a_decode_step(cuda_device):
    """Projection, append and attention one after the other, for a few steps, against the 64-bit forms."""
    heads, kv_heads, dim, page, hidden = 8, 2, 64, 16, 256
    g = torch.Generator().manual_seed(1)
    w = torch.randint(0, 256, ((heads + 2 * kv_heads) * dim, hidden // 2), generator=g).to(torch.uint8).to(cuda_device)
    scale = ((torch.rand((w.shape[0], hidden // 64), generator=g) + 0.5) * 0.01).to(BF16).to(cuda_device)
    cache = list(ref.make_cache(8, kv_heads, page, dim, E4M3, cuda_device))
    table = torch.tensor([[3, 1, 7], [6, 0, 2]], dtype=torch.int32, device=cuda_device)
    for step in range(4):
        x = torch.randn((2, hidden), generator=g).to(BF16).to(cuda_device)
        lens = torch.tensor([15 + step, 30 + step], dtype=torch.int32, device=cuda_device)
        qkv = xla_b200.dot_w4(x, w, scale)
        _check_dot(qkv, [x, w, scale, None, None], hidden)
        q, k_new, v_new = (t.reshape(2, 1, -1, dim).contiguous() for t in qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        _check_append([k_new, v_new, *cache, table, lens], None)
        _check_attention([q, *cache, table, lens])


def test_calls_on_a_side_stream_and_in_two_graphs(cuda_device):
    """Two captured steps share the workspace and the cache and are replayed with other lengths and inputs."""
    args = _attention_inputs(cuda_device, 8, 2, 128, 16, [400, 90], 1, E4M3, BF16)
    longest = args[6].clone()
    work = torch.empty(xla_b200.paged_attention_workspace_bytes(2, 1, 8, 2, 128), dtype=torch.int8, device=cuda_device)
    x, w, scale, _, _ = _dot_inputs(cuda_device, 2, 64, 256, 64, BF16, False, False)
    new = torch.randn((2, 1, 2, 128), device=cuda_device).to(BF16)
    sites, graphs, outs = [], [], []
    for _ in range(2):
        out, y = torch.empty_like(args[0]), torch.empty((2, 64), dtype=BF16, device=cuda_device)
        lse = torch.empty(out.shape[:3], device=cuda_device)
        calls = [xla_b200.DotW4Call([x, w, scale], [y]), xla_b200.KvCacheAppendCall([new, new, *args[1:]], args[1:5]),
                 xla_b200.PagedAttentionKv8Call(args, [out, lse, work], softmax_scale=128 ** -0.5, emit_lse=True)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for call in calls:
                call.run(stream.cuda_stream, 0)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for call in calls:
                call.execute(torch.cuda.current_stream().cuda_stream, 0)
        sites.append(calls)
        graphs.append(graph)
        outs.append((out, lse, y))
    for lens in ([400, 90], [1, 17], [33, 0], [399, 64]):
        args[6].copy_(torch.minimum(torch.tensor(lens, dtype=torch.int32, device=cuda_device), longest))
        args[0].normal_()
        x.normal_()
        new.normal_()
        want = [t.clone() for t in args[1:5]]
        fresh = torch.clamp(args[6], max=1)
        want = ref.append(new, new, *want, args[5], args[6], fresh)
        for graph, (out, lse, y) in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(args[1:5], want))
            _check_attention(args, [min(n, 1) for n in args[6].tolist()], out=(out, lse))
            _check_dot(y, [x, w, scale, None, None], 256)
    assert _status() == 0


def test_calls_side_by_side_on_two_streams(cuda_device):
    """Two attentions with their own workspaces at the same time give what each gives alone."""
    a = _attention_inputs(cuda_device, 16, 2, 128, 64, [9000, 300], 1, E4M3, BF16, seed=1)
    b = _attention_inputs(cuda_device, 8, 8, 64, 16, [5000], 2, S8, F16, seed=2)
    alone = [xla_b200.paged_attention_kv8(*t) for t in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, (stream, t) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(stream):
                got[i].append(xla_b200.paged_attention_kv8(*t))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(alone[i], t) for t in got[i])
