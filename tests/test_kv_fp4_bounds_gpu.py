"""The 4-bit K/V pool in the bounds-checking build: what it reports, and that scratch and workspaces keep their guard zones."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

_CHILD = r"""
import torch
from minisglang_rdna4_b200 import ops
from minisglang_rdna4_b200.ops import cuda as K

assert K.bounds_checks_enabled() and K.bounds_report() == []
ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
pages, hk, dim = 40, 2, 128
cache = torch.zeros(2, pages, hk, 1, 18 * dim, dtype=torch.uint8, device="cuda")
weights = torch.zeros(2, pages, hk, 16, device="cuda")
k, v = (torch.randn(4, hk, dim, device="cuda").bfloat16() for _ in range(2))
# rows without a slot are ordinary; one behind the pool is not
ops.store_kv_fp4(k, v, cache[0], ints([3, -1, 5, -1]))
assert K.bounds_report() == []
ops.store_kv_fp4(k, v, cache[0], ints([3, -1, 16 * pages, 7]))
rep = K.bounds_report()
assert rep and all(r.startswith("kv_fp4.cu:") and r.endswith("value 640 limit 640") for r in rep), rep
ops.load_kv_fp4(cache[0], ints([-1, 16 * pages + 2, 7]))
rep = K.bounds_report()
assert rep and all(r.startswith("kv_fp4.cu:") and r.endswith("value 642 limit 640") for r in rep), rep
# new pages of an eviction
table, lens = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10), ints([150, 30])
ops.evict_kv_fp4(cache, weights, table, lens, ints([[20, 21], [22, 23]]), 32, 5)
assert K.bounds_report() == []
ops.evict_kv_fp4(cache, weights, table, lens, ints([[20, 77], [22, 23]]), 32, 5)
rep = K.bounds_report()
assert rep and all(r.startswith("kv_fp4.cu:") and r.endswith("value 77 limit 40") for r in rep), rep
# all forms of attention: nothing to report, guard zones whole
for window in (0, 40):
    for news in ([1, 1], [5, 30], [150, 30]):
        q = torch.randn(sum(news), 8, dim, device="cuda").bfloat16()
        cu = ints([0, news[0], sum(news)])
        ops.paged_attention_fp4(q, cache[0], table, cu, lens, 0.1, window=window, max_q=max(news), weights=weights[0])
        plan = ops.prefill_plan_fp4(q, cache[0], cu.cpu().numpy(), lens.cpu().numpy(), window)
        if news[0] == 150:
            assert plan is not None
            for stream in [torch.cuda.Stream() for _ in range(6)]:
                stream.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(stream):
                    ops.paged_attention_fp4(q, cache[0], table, cu, lens, 0.1, window=window, max_q=150, plan=plan)
                torch.cuda.current_stream().wait_stream(stream)
torch.cuda.synchronize()
assert K.bounds_report() == [] and K.verify_workspaces() == []
assert len(K._TC_SCRATCH) == K.TC_SCRATCH_SETS
assert sum(name.startswith("prefill") for name in K._GUARDED) == 2 * K.TC_SCRATCH_SETS, list(K._GUARDED)
assert K.attn_status() == 0
# a page behind the pool in a request's table is named too, and read as the pool's last
ops.paged_attention_fp4(q[:1], cache[0], ints([[0, 41]]), ints([0, 1]), ints([20]), 0.1, max_q=1)
rep = K.bounds_report()
assert rep and all(r.startswith("attention_fp4.cu:") and r.endswith("value 41 limit 40") for r in rep), rep
print("BOUNDS-OK")
"""


def test_bounds_checking_build():
    from minisglang_rdna4_b200.ops import _lib

    if not os.path.exists(_lib.CHECKED_LIB_PATH):
        from minisglang_rdna4_b200 import build

        build.build_cuda(checked=True)
    out = subprocess.run([sys.executable, "-c", _CHILD], capture_output=True, text=True, env=dict(os.environ, MSGL_CHECK_BOUNDS="1"),
                         timeout=600, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert out.returncode == 0 and "BOUNDS-OK" in out.stdout, out.stdout[-2000:] + out.stderr[-4000:]
