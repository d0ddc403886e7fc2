"""What the calls of a drafted round refuse, and how they cut their work, on the CPU: the kernel set with its device checks and its
library replaced by recorders."""

import ctypes
import random

import pytest
import torch

from ampere_kv_engine_amd.csrc import build
from ampere_kv_engine_amd.kernels import hip_rounds
from ampere_kv_engine_amd.kernels.hip import HipKernels, KernelError

I32 = torch.int32


class Recorder(HipKernels):
    """Takes host tensors; calls end in `calls` instead of in a library."""

    def __init__(self):
        self.device, self.compute_units, self.calls = torch.device("cpu"), 256, []
        self._place_most = 4096

    def _dense(self, t, name, dtype=None, shape=None):
        if not isinstance(t, torch.Tensor):
            raise KernelError(f"{name} must be a tensor")
        if not t.is_contiguous():
            raise KernelError(f"{name} must be contiguous")
        if dtype is not None and t.dtype != dtype:
            raise KernelError(f"{name} must be {dtype}")
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise KernelError(f"{name} must have shape {tuple(shape)}")
        return t

    def _placed(self, t, name):
        pass

    def _stream(self):
        return None

    def _shared_prefix_entry(self, head_dim):
        return lambda *arguments: self.calls.append(arguments) or 0

    def _rounds(self):
        recorder = self

        class Library:
            def akv_verify_workspace(self, requests, places, vocab):
                return -1 if places > 64 or vocab > 262144 or requests > 65535 else 1024

            def akv_verify_drafts(self, *arguments):
                recorder.calls.append(arguments)
                return 0

            akv_place_tokens = akv_verify_drafts

        return Library()


def attention(**changes):
    """A call that is taken, with `changes`."""
    q = torch.zeros(5, 8 * 64)
    arguments = dict(q=q, k_pages=torch.zeros(12, 2, 16, 64), v_pages=torch.zeros(12, 2, 64, 16), block_table=torch.zeros(3, 6, dtype=I32),
                     q_start=torch.tensor([0, 1, 3, 5], dtype=I32), seq_lens=torch.tensor([40, 60, 70], dtype=I32), shared=32, q_heads=8,
                     kv_heads=2, head_dim=64, scale=0.125, out=torch.zeros_like(q), max_seq_len=96, max_new_tokens=2)
    arguments.update(changes)
    return arguments


def test_a_good_attention_call_is_made():
    kernels = Recorder()
    kernels.attention_shared_prefix(**attention())
    kernels.attention_shared_prefix(**attention(rows=torch.tensor([7, 0, 2], dtype=I32), block_table=torch.zeros(9, 6, dtype=I32)))
    kernels.attention_shared_prefix(**attention(shared=0))
    assert len(kernels.calls) == 3


@pytest.mark.parametrize("changes", [
    dict(q=torch.zeros(5, 8 * 64).double()), dict(q=torch.zeros(5, 8 * 64).half()), dict(q=torch.zeros(5, 500)), dict(q=torch.zeros(10, 512)[::2]),
    dict(out=torch.zeros(5, 512, dtype=torch.bfloat16)), dict(out=torch.zeros(4, 512)),
    dict(k_pages=torch.zeros(12, 2, 16, 32)), dict(k_pages=torch.zeros(12, 2, 16, 64, dtype=torch.bfloat16)), dict(v_pages=torch.zeros(12, 2, 16, 64)),
    dict(k_pages=torch.zeros(12, 2, 4, 64), v_pages=torch.zeros(12, 2, 64, 4)), dict(k_pages=torch.zeros(12, 2, 24, 64), v_pages=torch.zeros(12, 2, 64, 24)),
    dict(k_pages=torch.zeros(0, 2, 16, 64), v_pages=torch.zeros(0, 2, 64, 16)),
    dict(block_table=torch.zeros(3, 6)), dict(block_table=torch.zeros(2, 6, dtype=I32)), dict(block_table=torch.zeros(18, dtype=I32)),
    dict(block_table=torch.zeros(3, 5, dtype=I32)), dict(q_start=torch.zeros(3, dtype=I32)), dict(q_start=torch.zeros(4, dtype=torch.int64)),
    dict(seq_lens=torch.zeros(3)), dict(rows=torch.zeros(2, dtype=I32)), dict(shared=-16), dict(shared=40), dict(shared=96), dict(max_seq_len=32),
    dict(max_seq_len=97), dict(max_new_tokens=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
    dict(q_heads=7), dict(kv_heads=3), dict(head_dim=60), dict(head_dim=272),
], ids=str)
def test_attention_refuses(changes):
    kernels = Recorder()
    with pytest.raises(KernelError):
        kernels.attention_shared_prefix(**attention(**changes))
    assert not kernels.calls


def test_attention_refuses_odd_addresses():
    kernels = Recorder()
    with pytest.raises(KernelError, match="16-byte"):
        kernels.attention_shared_prefix(**attention(q=torch.zeros(5 * 512 + 1)[1:].view(5, 512)))


def test_nothing_to_attend_to_is_no_call():
    kernels = Recorder()
    kernels.attention_shared_prefix(**attention(q=torch.zeros(0, 512), out=torch.zeros(0, 512)))
    assert not kernels.calls


def verification(**changes):
    arguments = dict(logits=torch.zeros(7, 100), tokens=torch.zeros(7, dtype=I32), q_start=torch.zeros(4, dtype=I32), temperature=torch.zeros(3),
                     uniforms=torch.zeros(3, 4), kept=torch.zeros(3, dtype=I32), chosen=torch.zeros(3, 4, dtype=I32),
                     draft_logits=torch.zeros(3, 3, 100))
    arguments.update(changes)
    return arguments


def test_good_verifications_are_made():
    kernels = Recorder()
    kernels.verify_drafts(**verification())
    kernels.verify_drafts(**verification(draft_logits=None))
    kernels.verify_drafts(**verification(draft_logits=torch.zeros(3, 3, 100).transpose(0, 1).contiguous().transpose(0, 1)))
    kernels.verify_drafts(**verification(draft_logits=torch.zeros(3, 1, 100).expand(3, 3, 100)))
    kernels.verify_drafts(**verification(uniforms=torch.zeros(3, 1), chosen=torch.zeros(3, 1, dtype=I32), draft_logits=torch.zeros(3, 0, 100)))
    assert len(kernels.calls) == 5 and kernels.calls[2][10:12] == (100, 300) and kernels.calls[3][10:12] == (100, 0)


@pytest.mark.parametrize("changes", [
    dict(logits=torch.zeros(7, 100).double()), dict(logits=torch.zeros(700)), dict(logits=torch.zeros(7, 200)[:, :100]), dict(tokens=torch.zeros(6, dtype=I32)),
    dict(tokens=torch.zeros(7, dtype=torch.int64)), dict(q_start=torch.zeros(3, dtype=I32)), dict(temperature=torch.zeros(2)),
    dict(temperature=torch.zeros(3).double()), dict(uniforms=torch.zeros(12)), dict(uniforms=torch.zeros(3, 8)[:, ::2]), dict(kept=torch.zeros(3)),
    dict(chosen=torch.zeros(3, 5, dtype=I32)), dict(draft_logits=torch.zeros(3, 4, 100)), dict(draft_logits=torch.zeros(3, 3, 99)),
    dict(draft_logits=torch.zeros(3, 3, 200)[:, :, ::2]), dict(draft_logits=torch.zeros(3, 3, 100).bfloat16()),
    dict(uniforms=torch.zeros(3, 65), chosen=torch.zeros(3, 65, dtype=I32), draft_logits=None),
    dict(logits=torch.zeros(1, 600000), tokens=torch.zeros(1, dtype=I32), draft_logits=None),
], ids=lambda c: ",".join(f"{k}{tuple(v.shape) if v is not None else None}{v.dtype if v is not None else ''}" for k, v in c.items()))
def test_verification_refuses(changes):
    kernels = Recorder()
    with pytest.raises(KernelError):
        kernels.verify_drafts(**verification(**changes))
    assert not kernels.calls


def layout(**changes):
    vector = lambda n: torch.zeros(n, dtype=I32)
    arguments = dict(lengths=vector(3), counts=vector(3), held=vector(3), free_pages=vector(9), cursor=vector(1), table=torch.zeros(3, 4, dtype=I32),
                     page_size=16, q_start=vector(4), seq_lens=vector(3), held_after=vector(3), cursor_after=vector(1), positions=vector(5),
                     seq_of_token=vector(5), slot_map=vector(5), status=vector(1))
    arguments.update(changes)
    return arguments


def test_good_layouts_are_made():
    kernels = Recorder()
    kernels.place_tokens(**layout())
    kernels.place_tokens(**layout(rows=torch.zeros(3, dtype=I32), prefix_pages=torch.zeros(2, dtype=I32), table=torch.zeros(1, 4, dtype=I32)))
    kernels.place_tokens(**layout(positions=torch.zeros(0, dtype=I32), seq_of_token=torch.zeros(0, dtype=I32), slot_map=torch.zeros(0, dtype=I32)))
    assert len(kernels.calls) == 3


@pytest.mark.parametrize("name", ["counts", "held", "cursor", "q_start", "seq_lens", "held_after", "cursor_after", "seq_of_token", "slot_map", "status"])
@pytest.mark.parametrize("how", ["long", "int64", "strided", "matrix"])
def test_layout_refuses_vectors(name, how):
    kernels = Recorder()
    good = layout()[name]
    bad = dict(long=torch.zeros(len(good) + 1, dtype=I32), int64=good.long(), strided=torch.zeros(2 * max(len(good), 2), dtype=I32)[::2][:len(good)],
               matrix=good[None])[how]
    if how == "strided" and len(good) == 1:
        return              # (a single number has no stride)
    with pytest.raises(KernelError):
        kernels.place_tokens(**layout(**{name: bad}))
    assert not kernels.calls


@pytest.mark.parametrize("changes", [dict(table=torch.zeros(2, 4, dtype=I32)), dict(table=torch.zeros(12, dtype=I32)), dict(table=torch.zeros(3, 4)),
                                     dict(rows=torch.zeros(2, dtype=I32)), dict(page_size=0), dict(page_size=-16), dict(page_size=1.5),
                                     dict(prefix_pages=torch.zeros(2))], ids=str)
def test_layout_refuses(changes):
    kernels = Recorder()
    with pytest.raises(KernelError):
        kernels.place_tokens(**layout(**changes))
    assert not kernels.calls


def test_layout_refuses_more_requests_than_it_takes():
    kernels = Recorder()
    n = 4097
    vector = lambda: torch.zeros(n, dtype=I32)
    with pytest.raises(KernelError, match="4096"):
        kernels.place_tokens(**layout(lengths=vector(), counts=vector(), held=vector(), seq_lens=vector(), held_after=vector(),
                                      q_start=torch.zeros(n + 1, dtype=I32), table=torch.zeros(n, 1, dtype=I32)))


def test_spans_that_overlap():
    """The entries' check of what memory their operands share, by itself."""
    lib = ctypes.CDLL(build.ensure_rounds())

    def shared(written, *spans):
        begins = (ctypes.c_void_p * len(spans))(*(begin or None for begin, _ in spans))
        sizes = (ctypes.c_long * len(spans))(*(size for _, size in spans))
        return lib.akv_shared_spans(begins, sizes, written, len(spans))

    assert shared(1, (100, 20), (120, 4), (96, 4), (300, 0)) == 0
    assert shared(1, (100, 20), (119, 4)) == -(1000 + 1)
    assert shared(1, (100, 20), (200, 8), (90, 11)) == -(1000 + 2)
    assert shared(1, (100, 20), (50, 500)) == -(1000 + 1)
    assert shared(2, (100, 20), (200, 20), (300, 4), (210, 1)) == -(1000 + 64 + 3)
    assert shared(1, (100, 20), (200, 40), (210, 40)) == 0           # (what is only read may overlap)
    assert shared(1, (100, 0), (100, 0)) == 0 and shared(1, (100, 20), (110, 0)) == 0 and shared(1, (100, 20), (0, 500)) == 0


def test_what_shares_memory_is_named():
    kernels = Recorder()
    kernels._shared_prefix_entry = lambda head_dim: lambda *arguments: -(1000 + 2)
    with pytest.raises(KernelError, match="out and k_pages share memory"):
        kernels.attention_shared_prefix(**attention())
    with pytest.raises(KernelError, match="dtype not supported"):
        kernels._check_spans(-1, "this", ())


def test_segments_cover_the_keys():
    rng = random.Random(3)
    for _ in range(3000):
        requests, kv_heads, rows = rng.choice((1, 2, 7, 64, 500)), rng.choice((1, 2, 8, 32)), rng.choice((1, 4, 40, 900, 20000))
        most, shared = rng.choice((1, 5, 127, 128, 129, 2000, 131072)), rng.choice((0, 8, 16, 512, 8192, 131072))
        own_segments, own_keys = hip_rounds.cut_own(requests, min(rows, 600), kv_heads, most, 256)
        assert own_segments <= 256 and own_keys % 32 == 0 and (own_segments - 1) * own_keys < most <= own_segments * own_keys
        for columns in (32, 256):
            segments, keys = hip_rounds.cut_prefix(columns, rows, kv_heads, shared, 256, rng.random() < 0.5)
            assert keys % 32 == 0 and segments * keys >= shared and (segments == 0 if shared == 0 else (segments - 1) * keys < shared)
            assert segments + own_segments <= 512


def test_wide_tiles_are_for_many_columns_of_long_prompts():
    assert not hip_rounds.wide_tiles(32, 8, 8192, 256) and hip_rounds.wide_tiles(256, 8, 32768, 256) and not hip_rounds.wide_tiles(64, 8, 1 << 20, 256)
    assert hip_rounds.wide_tiles_fit(128, 16, torch.bfloat16) and not hip_rounds.wide_tiles_fit(128, 8, torch.bfloat16)
    assert not hip_rounds.wide_tiles_fit(128, 16, torch.float32) and not hip_rounds.wide_tiles_fit(96, 16, torch.bfloat16)


def test_the_wide_kernel_keeps_its_registers():
    """A spilled register in its loop would be a wait for every load on its way, and more than 256 leave its eight waves no room."""
    import test_kernel_code_host as code
    import tempfile
    for dim in (64, 128):
        with tempfile.TemporaryDirectory() as folder:
            facts = code._kernel_facts(code._device_codes(build.shared_prefix_library_path(dim), folder))
        found = [fact for name, fact in facts.items() if "wide_prefix_kernel" in name]
        assert len(found) == 1 and found[0]["vgpr_count"] <= 256 and found[0]["vgpr_spill_count"] == 0, found
