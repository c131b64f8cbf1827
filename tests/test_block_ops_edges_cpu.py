"""Block operators without a GPU: what the package needs of torch, and calls that are refused before a launch."""
import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_package_imports_without_cuda_in_torch():
    """A torch built without CUDA has no ``_cuda_getCurrentRawStream``: registries and oracles load there all the same,
    and the stream comes from the public call."""
    code = """
import torch
del torch._C._cuda_getCurrentRawStream
import segment_anything_fast_b200
from segment_anything_fast_b200 import ops
class Stream:
    cuda_stream = 77
torch.cuda.current_device = lambda: 1
torch.cuda.current_stream = lambda dev: Stream if dev == 1 else None
assert ops._stream() == 77
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_grouped_warps_leave_their_roles_together():
    """A wait that runs out may do so for some lanes of a warp only.  In the roles that a whole warp walks, no lane may act
    on its own answer (the others would meet it in elect.sync or __syncwarp and wait for good): a wait's result is only
    kept, what is issued asks for it behind the election, and the way out is a vote."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "segment_anything_fast_b200", "csrc", "gemm_grouped.cu")).read())
    uses = re.findall(r"[^;{}]*\bwarp_wait\([^;]*;", text.split("tile_list", 1)[1])
    assert len(uses) == 6                                # W, gathered rows, twice the MMA warp's two
    for use in uses:
        assert re.fullmatch(r"ok = (ok && )?warp_wait\([^;]*\);", use.strip()), use
    assert text.count("if (elect_one() && ok)") == 4 and "__activemask" not in text
    assert len(re.findall(r"ok = __all_sync\(0xffffffffu, ok\)", text)) == 4
    for role in re.split(r"\bok = true;", text)[1:]:
        role = role.split("warp ==", 1)[0]
        if "warp_wait(" in role:
            assert role.rindex("__all_sync") > role.rindex("warp_wait(")
            assert not re.search(r"if \(!ok\)|\(!\(ok = warp_wait", role)
