"""What the calls of a drafted round promise at their limits, on the CPU: the library replaced by a recorder."""

import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from ampere_kv_engine_amd.csrc import build
from ampere_kv_engine_amd.kernels import hip_rounds
from ampere_kv_engine_amd.kernels.hip import KernelError
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


def test_partial_sums_stay_within_their_room_whatever_the_bound():
    """A call over a long table, as it is recorded, brings its bound and not its lengths."""
    for requests, new, heads, dim in ((64, 5, 64, 128), (64, 1, 32, 128), (500, 1, 32, 128), (500, 5, 64, 256), (1, 1, 16, 64)):
        tokens = requests * new
        of_segment = 4 * tokens * heads * (dim + 2)
        for most in (1, 500, 2048, 32768, 131072, 1 << 20):
            segments, keys = hip_rounds.cut_own(requests, new * heads // 8, 8, most, 256, of_segment)
            assert segments * of_segment <= max(hip_rounds.OWN_ROOM, 8 * of_segment) and segments <= 256
            assert keys % 128 == 0 and (segments - 1) * keys < most <= segments * keys
            if most <= 2048:      # (bounds that are near the lengths: cut by what the blocks do)
                assert (segments, keys) == hip_rounds.cut_own(requests, new * heads // 8, 8, most, 256)


def test_the_call_takes_its_room_into_account():
    q = torch.zeros(320, 64 * 16)
    kernels = Recorder()
    arguments = attention(q=q, out=torch.zeros_like(q), q_heads=64, kv_heads=8, head_dim=16, k_pages=torch.zeros(2, 8, 16, 16), v_pages=torch.zeros(2, 8, 16, 16),
                          block_table=torch.zeros(3, 1 << 16, dtype=torch.int32), max_seq_len=1 << 20, max_new_tokens=5, shared=0)
    hip_rounds_room, hip_rounds.OWN_ROOM = hip_rounds.OWN_ROOM, 64 << 20
    try:
        kernels.attention_shared_prefix(**arguments)
    finally:
        hip_rounds.OWN_ROOM = hip_rounds_room
    own_segments = kernels.calls[0][-4]
    assert own_segments * 4 * 320 * 64 * 18 <= 64 << 20 and own_segments >= 40


def test_attention_refuses_pages_of_a_prompt_that_are_too_few():
    ints = lambda *shape, dtype=torch.int32: torch.zeros(*shape, dtype=dtype)
    kernels = Recorder()
    kernels.attention_shared_prefix(**attention(prefix_pages=ints(2)))          # 32 shared tokens, pages of 16
    kernels.attention_shared_prefix(**attention(prefix_pages=ints(5)))
    kernels.attention_shared_prefix(**attention(prefix_pages=ints(0), shared=0))
    assert len(kernels.calls) == 3
    for pages in (ints(1), ints(2, dtype=torch.int64), ints(2, 1), ints(4)[::2]):
        with pytest.raises(KernelError):
            kernels.attention_shared_prefix(**attention(prefix_pages=pages))
    assert len(kernels.calls) == 3


def test_bounds_beyond_31_bits_are_no_bounds():
    """A table of pages so long that its width in tokens does not fit the lengths' type."""
    q = torch.zeros(5, 16)
    kernels = Recorder()
    kernels.attention_shared_prefix(**attention(q=q, out=torch.zeros_like(q), q_heads=1, kv_heads=1, head_dim=16, k_pages=torch.zeros(1, 1, 1 << 20, 16),
                                                v_pages=torch.zeros(1, 1, 16, 1 << 20), block_table=torch.zeros(3, 4097, dtype=torch.int32),
                                                shared=1 << 20, max_seq_len=1 << 32, max_new_tokens=1 << 40))
    max_own, max_new, _, _, own_segments, own_keys = kernels.calls[0][-8:-2]
    assert max_own == (1 << 30) - (1 << 20) and max_new == 5
    assert own_segments <= 256 and own_segments * own_keys >= max_own and (1 << 30) + own_keys < 2 ** 31
