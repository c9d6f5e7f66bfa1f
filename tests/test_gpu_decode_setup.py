"""The device set-up of the decode-step operators, each case in a process that has done nothing else."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

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
""", B200SD_LIBRARY=os.path.join(ROOT, "xla_b200", "lib", "libb200_scaled_dot_tuning.so"), B200SD_FAIL_DECODE_SETUP="1")


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
