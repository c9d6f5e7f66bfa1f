"""What the decode-step calls accept and refuse, without a device: call frames at the instantiate stage, the C entry
points' checks, and the plain 64-bit forms that the device tests compare with."""
import ctypes as C
import threading

import pytest
import torch

import decode_reference as ref
import xla_b200
from xla_b200 import _native
from xla_b200.scaled_dot import BF16, F16, F32, F8E4M3FN, F8E5M2, F64, S4, S8, S32, U4, U8, Buffer, FfiCall, XlaFfiError

INVALID, UNIMPLEMENTED = 3, 12


def _refused(status, make, *args, **kw):
    with pytest.raises(XlaFfiError) as e:
        make(*args, **kw).instantiate()
    assert e.value.code == status, str(e.value)


def _dot(m=4, n=48, k=256, group=64, x=BF16, w=U8, s=BF16, d=None, zero=None, bias=None, weight_type=S4, wk=None, groups=None, workspace=False, want_bias=None):
    ops = [Buffer(x, (m, k)), Buffer(w, (n, k // 2 if wk is None else wk)), Buffer(s, (n, k // group if groups is None else groups))]
    ops += [b for b in (zero, bias) if b is not None]
    res = [Buffer(x if d is None else d, (m, n))] + ([Buffer(S8, (64,))] if workspace else [])
    return xla_b200.DotW4Call(ops, res, weight_type=weight_type, bias=bias is not None if want_bias is None else want_bias)


def test_dot_w4_frames():
    for kw in (dict(), dict(x=F16, s=F32), dict(d=F32), dict(w=S8), dict(m=1, n=1, k=32, group=32), dict(m=64), dict(m=0), dict(group=256), dict(workspace=True),
               dict(weight_type=U4, zero=Buffer(U8, (48, 4))), dict(bias=Buffer(F32, (48,)))):
        _dot(**kw).instantiate()
    for kw in (dict(x=F32), dict(s=F64), dict(d=F16), dict(w=S32), dict(wk=100), dict(groups=3), dict(groups=0), dict(k=96, group=48), dict(group=16), dict(k=64 * 5, groups=1),
               dict(weight_type=U4), dict(zero=Buffer(U8, (48, 4))), dict(weight_type=U4, zero=Buffer(S32, (48, 4))), dict(weight_type=U4, zero=Buffer(U8, (48, 8))),
               dict(weight_type=U8), dict(bias=Buffer(BF16, (47,))), dict(bias=Buffer(S32, (48,))), dict(want_bias=True), dict(n=0)):
        _refused(INVALID, _dot, **kw)
    _refused(UNIMPLEMENTED, _dot, m=65)
    _refused(UNIMPLEMENTED, lambda: FfiCall("b200$dot$w4", [Buffer(BF16, (4, 64)), Buffer(U8, (8, 32)), Buffer(BF16, (8, 1))], [Buffer(BF16, (4, 8))], {"epilogue": ("i32", 4)}))
    _refused(INVALID, lambda: FfiCall("b200$dot$w4", [Buffer(BF16, (4, 64))], [Buffer(BF16, (4, 8))], {}))


def _cache(pages=9, kv_heads=2, page=16, dim=64, batch=3, width=4, code=F8E4M3FN, v=None, scale=F32, table=S32, lens=S32, new_lens=False):
    shape = (pages, kv_heads, page, dim)
    ops = [Buffer(code, shape), Buffer(code if v is None else v, shape), Buffer(scale, (pages, kv_heads)), Buffer(F32, (pages, kv_heads)),
           Buffer(table, (batch, width)), Buffer(lens, (batch,))]
    return ops + ([Buffer(S32, (batch,))] if new_lens else [])


def _append(new=(3, 5, 2, 64), dtype=BF16, v_dtype=None, results=None, **kw):
    cache = _cache(**kw)
    return xla_b200.KvCacheAppendCall([Buffer(dtype, new), Buffer(dtype if v_dtype is None else v_dtype, new)] + cache, cache[:4] if results is None else results)


def test_append_frames():
    for kw in (dict(), dict(dtype=F16), dict(code=S8), dict(code=F8E5M2), dict(new_lens=True), dict(page=128), dict(pages=0, width=0), dict(new=(3, 0, 2, 64)), dict(new=(0, 5, 2, 64), batch=0),
               dict(new=(3, 5000, 2, 64)), dict(dim=16, new=(3, 1, 2, 16)), dict(dim=256, new=(3, 1, 2, 256))):
        _append(**kw).instantiate()
    other = [Buffer(b.dtype, b.dims, 4096) for b in _cache()[:4]]
    for kw in (dict(dtype=F32), dict(v_dtype=F16), dict(code=BF16), dict(v=S8), dict(scale=BF16), dict(table=F32), dict(lens=F32), dict(page=24), dict(page=256),
               dict(dim=40, new=(3, 1, 2, 40)), dict(dim=272, new=(3, 1, 2, 272)), dict(new=(3, 5, 3, 64)), dict(new=(2, 5, 2, 64)), dict(new=(3, 5, 2, 32)),
               dict(results=_cache()[:3]), dict(results=_cache(code=S8)[:4])):
        _refused(INVALID, _append, **kw)
    _refused(UNIMPLEMENTED, _append, new=(5000, 1, 2, 64), batch=5000)
    # At the execute stage the results have to be the operands' own buffers; nothing is launched before that is seen.
    call = _append(results=other)
    with pytest.raises(XlaFfiError) as e:
        call.execute()
    assert e.value.code == INVALID and "output_to_operand_aliasing" in str(e.value)


def _attend(q=(3, 1, 4, 64), dtype=BF16, out=None, out_dtype=None, lse=None, emit_lse=False, scale=0.125, window=0, workspace=True, **kw):
    res = [Buffer(dtype if out_dtype is None else out_dtype, q if out is None else out)] + ([lse] if lse is not None else []) + ([Buffer(S8, (1 << 20,))] if workspace else [])
    return xla_b200.PagedAttentionKv8Call([Buffer(dtype, q)] + _cache(**kw), res, softmax_scale=scale, window=window, emit_lse=emit_lse)


def test_attention_frames():
    for kw in (dict(), dict(dtype=F16), dict(code=S8), dict(new_lens=True), dict(q=(3, 64, 4, 64)), dict(q=(3, 1, 2, 64)), dict(q=(3, 1, 34, 64)), dict(window=7), dict(scale=-2.0),
               dict(emit_lse=True, lse=Buffer(F32, (3, 1, 4))), dict(pages=0, width=0), dict(q=(0, 1, 4, 64), batch=0)):
        _attend(**kw).instantiate()
    for kw in (dict(dtype=F32), dict(out_dtype=F32), dict(out=(3, 1, 4, 32)), dict(q=(3, 1, 5, 64)), dict(q=(3, 1, 1, 64)), dict(q=(3, 1, 4, 32)), dict(q=(2, 1, 4, 64)), dict(window=-1),
               dict(scale=float("inf")), dict(scale=float("nan")), dict(emit_lse=True), dict(lse=Buffer(F32, (3, 1, 4))), dict(emit_lse=True, lse=Buffer(BF16, (3, 1, 4))),
               dict(workspace=False), dict(code=BF16), dict(page=48), dict(width=1 << 27), dict(pages=1 << 31)):
        _refused(INVALID, _attend, **kw)
    _refused(UNIMPLEMENTED, _attend, q=(3, 65, 4, 64))
    _refused(UNIMPLEMENTED, _attend, q=(4096, 64, 4096, 256), dim=256, batch=4096, kv_heads=512)     # 2^27 items; 2^26 are the most
    _attend(q=(4096, 64, 4096, 64), batch=4096, kv_heads=512).instantiate()
    _refused(INVALID, lambda: FfiCall("b200$paged_attention$kv8", [Buffer(BF16, (3, 1, 4, 64))] + _cache(), [Buffer(BF16, (3, 1, 4, 64)), Buffer(S8, (64,))], {}))


def test_c_entry_points_check_pointers_and_sizes():
    """Null and misaligned pointers and short workspaces are refused before a device is looked at."""
    err = C.create_string_buffer(256)

    def rc(name, args, check=False):
        fn = getattr(_native.product, "b200sd_" + ("check_" if check else "") + name)
        return fn(C.byref(args), err, len(err)) if check else fn(C.byref(args), None, err, len(err))

    def dot(**kw):
        a = _native.DotW4Args(m=2, n=8, k=64, group=32, x_dtype=BF16, weight_type=S4, scale_dtype=F32, d_dtype=F32, x=4096, w=4096, scale=4096, d=4096)
        a.struct_size = C.sizeof(a)
        for key, v in kw.items():
            setattr(a, key, v)
        return a

    assert rc("dot_w4", dot(), check=True) == 0
    for kw in (dict(x=None), dict(w=None), dict(scale=None), dict(d=None), dict(x=4104), dict(w=4097), dict(scale=4098), dict(d=4098), dict(weight_type=U4), dict(epilogue=1, bias_dtype=BF16),
               dict(epilogue=1, bias_dtype=F32, bias=4098), dict(struct_size=8), dict(m=-1), dict(k=1 << 25)):
        assert rc("dot_w4", dot(**kw)) == INVALID, kw
    base = dict(k_pages=4096, v_pages=4096, k_scale=4096, v_scale=4096, page_table=4096, seq_lens=4096, batch=2, new_tokens=1, kv_heads=2, head_dim=64, num_pages=8, page_tokens=16,
                table_width=4, cache_dtype=F8E4M3FN)

    def append(**kw):
        a = _native.KvCacheAppendArgs(**{**base, **dict(k_new=4096, v_new=4096, new_dtype=BF16), **kw})
        a.struct_size = kw.get("struct_size", C.sizeof(a))
        return a

    def attend(**kw):
        a = _native.PagedAttentionArgs(**{**base, **dict(q=4096, out=4096, heads=4, q_dtype=BF16, softmax_scale=1.0, workspace=4096, workspace_bytes=1 << 26), **kw})
        a.struct_size = kw.get("struct_size", C.sizeof(a))
        return a

    for name, make in (("kv_cache_append", append), ("paged_attention", attend)):
        assert rc(name, make(), check=True) == 0
        for kw in (dict(k_pages=None), dict(v_scale=None), dict(page_table=None), dict(seq_lens=None), dict(k_pages=4104), dict(v_scale=4098), dict(new_lens=4097), dict(struct_size=8), dict(num_pages=-1)):
            assert rc(name, make(**kw)) == INVALID, (name, kw)
    assert rc("kv_cache_append", append(k_new=None)) == INVALID and rc("kv_cache_append", append(v_new=4104)) == INVALID
    for kw in (dict(q=None), dict(out=None), dict(q=4104), dict(lse=4098), dict(workspace=None), dict(workspace=4104), dict(workspace_bytes=15)):
        assert rc("paged_attention", attend(**kw)) == INVALID, kw
    assert xla_b200.paged_attention_workspace_bytes(2, 1, 4, 2, 64) >= 16 and xla_b200.paged_attention_workspace_bytes(0, 1, 4, 2, 64) == 0


def test_functions_refuse_tensors_off_the_device_and_with_strides():
    x, w, s = torch.zeros((2, 64), dtype=torch.bfloat16), torch.zeros((8, 32), dtype=torch.uint8), torch.zeros((8, 1))
    with pytest.raises(XlaFfiError):
        xla_b200.dot_w4(x, w, s)
    with pytest.raises(ValueError):
        xla_b200.dot_w4(x[:, ::2], w[:, ::2], s)
    with pytest.raises(ValueError):
        xla_b200.dot_w4(x, w.t().contiguous().t(), s)


def test_a_call_site_that_is_given_more_operands_after_a_call():
    """The frame that a site keeps between calls is built again."""
    call = _dot()
    for want in ("null", "got 4"):
        with pytest.raises(XlaFfiError) as e:
            call.execute()
        assert e.value.code == INVALID and want in str(e.value)
        _native.mock.mockffi_call_add_arg(call._h, U8, None, 2, (C.c_int64 * 2)(48, 4))
    call.close()


# ---- the plain forms themselves ------------------------------------------------------------------
def test_plain_quantiser_is_torch_s():
    """Rounding in 64 bits equals torch's conversion from f32, at every code and halfway between them."""
    for dtype in (ref.E4M3, ref.E5M2):
        codes = torch.arange(256, dtype=torch.uint8).view(dtype).double()
        codes = torch.sort(codes[torch.isfinite(codes)]).values
        y = torch.cat([codes, (codes[1:] + codes[:-1]) / 2, codes * 1.0001, torch.tensor([1e-9, -1e-9, 1e6, -1e6])])
        want = torch.clamp(y, -ref.QMAX[dtype], ref.QMAX[dtype]).float().to(dtype)
        assert torch.equal(ref.quantise(y, dtype).double(), want.double())
    assert ref.quantise(torch.tensor([0.5, 1.5, -2.5, 127.5, -300.0, float("nan")], dtype=torch.float64), ref.S8).tolist() == [0, 2, -2, 127, -127, 0]


def test_plain_append_keeps_values_within_half_a_step():
    """What the cache stands for after an append is within half a step of the values (twice that for re-rounded ones)."""
    k, v, ks, vs = ref.make_cache(4, 2, 16, 16, ref.E4M3, "cpu")
    table = torch.tensor([[2, 1]], dtype=torch.int32)
    tokens = torch.randn(1, 20, 2, 16, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    cache = (k, v, ks, vs)
    for t in range(20):
        cache = ref.append(tokens[:, t:t + 1], tokens[:, t:t + 1], *cache, table, torch.tensor([t + 1], dtype=torch.int32))
    held = torch.cat([cache[0].double()[page] * cache[2].double()[page][:, None, None] for page in (2, 1)], 1)[:, :20]
    want = tokens[0].transpose(0, 1).double()
    assert bool(((held - want).abs() <= 2 * 2.0 ** -4 * want.abs() + 2.0 ** -8).all())
    assert all(torch.frexp(s)[0].eq(0.5).all() for s in (cache[2][1:3], cache[3][1:3]))


def test_plain_attention_against_torch():
    """The row-by-row form equals torch's attention with a mask."""
    k, v, ks, vs = ref.make_cache(3, 2, 16, 32, ref.S8, "cpu")
    table, lens = torch.tensor([[1, 0, 2]], dtype=torch.int32), torch.tensor([40], dtype=torch.int32)
    q = torch.randn(1, 4, 6, 32, generator=torch.Generator().manual_seed(0)).to(torch.float16)
    out, lse, _, _ = ref.attention(q, k, v, ks, vs, table, lens, window=10)
    full = [torch.cat([p.double()[i] * s.double()[i][:, None, None] for i in (1, 0, 2)], 1)[:, :40].repeat_interleave(3, 0) for p, s in ((k, ks), (v, vs))]
    at, here = torch.arange(40)[None], torch.arange(36, 40)[:, None]
    mask = (at <= here) & (at > here - 10)
    want = torch.nn.functional.scaled_dot_product_attention(q[0].transpose(0, 1).double(), *full, attn_mask=mask)
    assert torch.allclose(out[0].transpose(0, 1), want, atol=1e-12)
    scores = (q[0].transpose(0, 1).double() @ full[0].transpose(1, 2) * 32 ** -0.5).masked_fill(~mask, float("-inf"))
    assert torch.allclose(lse[0].t(), torch.logsumexp(scores, -1), atol=1e-12)


def test_threads_on_one_call_site_get_their_own_messages(monkeypatch):
    """Both calls have failed before either reads its message."""
    both, got = threading.Barrier(2), {}
    sites = {"first": _dot(zero=Buffer(U8, (48, 4))), "second": _dot(groups=3)}
    wants = {"first": "got 4", "second": "k / group"}
    execute = _native.mock.mockffi_call_execute

    def failing(handle, stream, device, *message):
        rc = execute(sites[threading.current_thread().name]._h, stream, device, *message)
        both.wait(10)
        return rc

    call = _dot()
    monkeypatch.setattr(_native.mock, "mockffi_call_execute", failing)

    def work():
        with pytest.raises(XlaFfiError) as e:
            call.execute()
        got[threading.current_thread().name] = str(e.value)

    threads = [threading.Thread(target=work, name=name) for name in ("first", "second")]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(wants[name] in got[name] for name in wants), got


def test_workspace_bytes_are_those_of_a_call_that_is_served():
    """Zero for what the call refuses or does nothing for, sizes whose products leave 64 bits among them."""
    size = xla_b200.paged_attention_workspace_bytes
    assert size(4096, 64, 4096, 1024, 128) > 0 and size(1, 1, 1, 1, 16) > 0
    base = dict(batch=2, new_tokens=1, heads=4, kv_heads=2, head_dim=64)
    for kw in (dict(batch=0), dict(new_tokens=0), dict(batch=-1), dict(new_tokens=-1), dict(batch=4097), dict(new_tokens=65), dict(heads=5), dict(heads=0), dict(heads=8192), dict(kv_heads=0),
               dict(heads=4096, kv_heads=2048), dict(head_dim=20), dict(head_dim=0), dict(head_dim=272), dict(new_tokens=2 ** 62), dict(heads=2 ** 62),
               dict(batch=4096, new_tokens=64, heads=4096, kv_heads=512, head_dim=256)):
        sizes = {**base, **kw}
        assert size(*sizes.values()) == 0, kw
