"""What the calls of a drafted round promise at their limits, on the CPU: the library replaced by a recorder."""

import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import torch

from ampere_kv_engine_amd.csrc import build
from test_rounds_host import Recorder, attention


def test_the_caller_says_whether_weights_are_rounded_once():
    """A batch that goes in wide tiles by its sizes, and the same call with weights in two parts."""
    pages = dict(k_pages=torch.zeros(4, 8, 512, 64, dtype=torch.bfloat16), v_pages=torch.zeros(4, 8, 64, 512, dtype=torch.bfloat16))
    q = torch.zeros(100, 16 * 64, dtype=torch.bfloat16)
    arguments = attention(q=q, out=torch.zeros_like(q), q_heads=16, kv_heads=8, shared=32768, max_seq_len=33000, max_new_tokens=50,
                          block_table=torch.zeros(3, 65, dtype=torch.int32), **pages)
    kernels = Recorder()
    kernels.attention_shared_prefix(**arguments)
    kernels.attention_shared_prefix(**arguments, two_part_weights=True)
    assert [call[-2] for call in kernels.calls] == [1, 0]
    kernels.wide_prefix_tiles = True
    kernels.attention_shared_prefix(**arguments, two_part_weights=True)
    assert kernels.calls[-1][-2] == 0


def test_every_head_size_compiles():
    """What is asserted of a head size when it is compiled (that a lane's dims of the join lie in one head) holds for all that are taken."""
    source = os.path.join(build.HERE, build.SHARED_PREFIX_SOURCE)

    def compiled(dim):
        return subprocess.run([build._hipcc(), *build.FLAGS, f"-DAKV_HEAD_DIM={dim}", "--cuda-host-only", "-fsyntax-only", source],
                              capture_output=True, text=True)

    with ThreadPoolExecutor(max_workers=8) as pool:
        for result in pool.map(compiled, range(16, 257, 16)):
            assert result.returncode == 0, result.stderr
