"""The device set-up of the decode-step operators and the end of their waits, each case in a process of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TUNING = os.path.join(ROOT, "xla_b200", "lib", "libb200_scaled_dot_tuning.so")
with_tuning_build = pytest.mark.skipif(not os.path.exists(TUNING), reason="the tuning build is not there (make tuning)")

COMMON = """
import ctypes as C
import torch
import xla_b200
from xla_b200 import _native
from xla_b200.scaled_dot import XlaFfiError
dev = torch.device("cuda:0")
err = C.create_string_buffer(512)
x = torch.randn((2, 256), device=dev).to(torch.bfloat16)
w, scale = torch.randint(0, 256, (64, 128), device=dev, dtype=torch.uint8), torch.rand((64, 4), device=dev)
q, new = torch.randn((1, 1, 4, 64), device=dev).to(torch.bfloat16), torch.randn((1, 1, 2, 64), device=dev).to(torch.bfloat16)
cache = [torch.zeros((3, 2, 16, 64), device=dev, dtype=torch.int8) for _ in range(2)] + [torch.ones((3, 2), device=dev) for _ in range(2)]
table, lens = torch.tensor([[2, 1]], device=dev, dtype=torch.int32), torch.tensor([17], device=dev, dtype=torch.int32)
"""


def _run(program, **env):
    done = subprocess.run([sys.executable, "-c", COMMON + program], cwd=ROOT, env={**os.environ, **env}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-2000:]


@with_tuning_build
def test_its_failure_leaves_the_other_calls_alone():
    _run("""
a = torch.ones((16, 64), device=dev).to(torch.float8_e4m3fn)
one = torch.ones((), device=dev)
for _ in range(2):
    d, _ = xla_b200.cublas_lt_matmul_f8(a, a.t().contiguous(), one, one, out_dtype=torch.bfloat16)
    assert bool((d == 64).all())
    xla_b200.kv_cache_append(new, new, *cache, table, lens)
    for call in (lambda: xla_b200.dot_w4(x, w, scale), lambda: xla_b200.paged_attention_kv8(q, *cache, table, lens)):
        try:
            call()
        except XlaFfiError as e:
            assert e.code == 13 and "made to fail" in str(e), e
        else:
            raise AssertionError("the set-up did not fail")
assert _native.product.b200sd_init_device(err, len(err)) == 0
assert _native.product.b200sd_init_decode_operators(err, len(err)) == 13
torch.cuda.synchronize()
""", B200SD_LIBRARY=TUNING, B200SD_FAIL_DECODE_SETUP="1")


@pytest.mark.parametrize("first", ["b200sd_init_decode_operators", "b200sd_init_device"])
def test_first_calls_into_a_graph(first):
    """After either set-up call the first launches may be captured ones."""
    _run(f"""
assert _native.product.{first}(err, len(err)) == 0, err.value
""" + """
y, out = torch.empty((2, 64), device=dev), torch.empty_like(q)
work = torch.empty(xla_b200.paged_attention_workspace_bytes(1, 1, 4, 2, 64), device=dev, dtype=torch.int8)
calls = [xla_b200.DotW4Call([x, w, scale], [y]), xla_b200.KvCacheAppendCall([new, new, *cache, table, lens], cache),
         xla_b200.PagedAttentionKv8Call([q, *cache, table, lens], [out, work], softmax_scale=0.125)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for call in calls:
        call.execute(torch.cuda.current_stream().cuda_stream, 0)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, xla_b200.dot_w4(x, w, scale, out_dtype=torch.float32))
assert torch.equal(out, xla_b200.paged_attention_kv8(q, *cache, table, lens)) and bool((out != 0).any())
assert xla_b200.device_status() == 0
""")


@with_tuning_build
def test_a_copy_that_does_not_come():
    """Its wait expires (20 ms in this build), the call ends and reports it, and the next one is right."""
    _run("""
import os
import sys
sys.path.insert(0, "tests")
import decode_reference as ref
g = torch.Generator().manual_seed(0)

def expires(call):
    os.environ["B200SD_LOSE_COPY"] = "1"
    call()
    del os.environ["B200SD_LOSE_COPY"]
    status = xla_b200.device_status()
    assert status == 128, status
    return call()

for m, n, k in ((8, 3000, 8192), (20, 100000, 640), (3, 40, 128), (64, 200, 1024)):
    x = torch.randn((m, k), generator=g).to(torch.bfloat16).to(dev)
    w = torch.randint(0, 256, (n, k // 2), generator=g).to(torch.uint8).to(dev)
    scale = torch.rand((n, k // 128), generator=g).to(dev)
    out = expires(lambda: xla_b200.dot_w4(x, w, scale, out_dtype=torch.float32))
    want, size = ref.dot(x, w, scale)
    assert bool(((out.double() - want).abs() <= (k + 4) * 2.0 ** -23 * size).all())
for heads, kv_heads, dim, lens in ((8, 2, 128, [9000, 40]), (32, 1, 64, [100, 300, 2]), (4, 2, 256, [5000])):
    pages = sum(-(-n // 16) for n in lens) + 1
    args = [torch.randn((len(lens), 1, heads, dim), generator=g).to(torch.bfloat16).to(dev), *ref.make_cache(pages, kv_heads, 16, dim, ref.E4M3, dev),
            ref.make_table(lens, 16, pages, dev), torch.tensor(lens, dtype=torch.int32, device=dev)]
    want = xla_b200.paged_attention_kv8(*args)
    assert xla_b200.device_status() == 0
    assert torch.equal(expires(lambda: xla_b200.paged_attention_kv8(*args)), want)
assert xla_b200.device_status() == 0
""", B200SD_LIBRARY=TUNING)
