"""What the calls of a drafted round promise at their limits, on the CPU: the library replaced by a recorder."""

import torch

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
