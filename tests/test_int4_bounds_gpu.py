"""4-bit pages on the bounds-checked kernel build (NE_DEBUG_BOUNDS=1): prompts whose expanded pages outnumber the cache's are valid and give what the ordinary build
gives; a bad entry of the real block table is still found.  No entry used here reaches memory that the test has not allocated."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

_SCRIPT = r"""
import hashlib, os, torch
from nanoengine_b200 import ops
from nanoengine_b200.ops import sm100
checked = os.environ["NE_DEBUG_BOUNDS"] == "1"
assert sm100.lib()._name.endswith("libne_kernels_dbg.so") == checked
sm100.clear_kernel_status()
assert sm100.debug_set_bounds(cache_rows=6 * 64, cache_pages=6, state_slots=0, experts=0) == checked
def call(hq, hkv, dim, new, ctx, table):
    g = torch.Generator().manual_seed(dim)
    kc, vc = (torch.cat([torch.randint(0, 256, (8, hkv, 64 * dim // 2), generator=g), torch.randint(72, 136, (8, hkv, 64 * dim // 32), generator=g)], -1).to(torch.uint8).cuda()
              for _ in range(2))
    q = torch.randn(sum(new), hq, dim, generator=g).to(torch.bfloat16).cuda()
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    return ops.gqa_attention_paged(q, kc, vc, torch.tensor(table, dtype=torch.int32, device="cuda"), cu, torch.tensor(ctx, dtype=torch.int32, device="cuda"), dim ** -0.5)
show = lambda t: hashlib.sha256(t.cpu().view(torch.uint8).numpy().tobytes()).hexdigest()[:16]
shared = [[2, 3, 4], [2, 3, 5], [2, 3, 1], [2, 3, 0]]                     # four sequences on two common pages: twelve expanded pages over a cache of six
for hq, hkv, dim, new in ((64, 4, 128, [40, 30, 50, 20]), (64, 4, 128, [150] * 4), (16, 4, 64, [150] * 4), (16, 2, 256, [100] * 4), (64, 4, 128, [1, 1, 1, 1])):
    out = call(hq, hkv, dim, new, [150 + 9 * i for i in range(4)], shared)
    torch.cuda.synchronize()
    assert sm100.kernel_status()[0] == 0, sm100.kernel_status()
    print("OUT", show(out))
if checked:
    for new in ([100], [1]):                                                # a page past the declared six, inside the eight that are there
        call(16, 4, 64, new, [190], [[1, 7, 2]])
        torch.cuda.synchronize()
        st = sm100.kernel_status()
        assert st[0] == 4 and st[4] == 7, st
        sm100.clear_kernel_status()
"""


def _run(checked):
    r = subprocess.run([sys.executable, "-c", _SCRIPT], env=dict(os.environ, NE_DEBUG_BOUNDS=checked), capture_output=True, text=True, timeout=280,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    return [line for line in r.stdout.splitlines() if line.startswith("OUT")]


def test_prompts_on_the_checked_build():
    from nanoengine_b200.build_native import build_kernels
    build_kernels(debug_bounds=True)                    # nothing to do when it was made from these sources
    want = _run("0")
    assert len(want) == 5 and _run("1") == want
