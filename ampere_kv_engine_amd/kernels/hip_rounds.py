"""Wrappers over the kernels of a round of drafted tokens: attention of requests that share a prompt (`csrc/shared_prefix.hip`, a
library per head size), the drafts' verification and the step's layout (`csrc/api_rounds.h`).  `HipKernels` inherits them.

They take the requests' lengths as they lie on the device and read nothing back, so that a round can follow the one before -
whose number of kept tokens no host has seen - or be recorded.  The host gives bounds (`max_seq_len`, `max_new_tokens`, the sizes of
the outputs); what a kernel finds outside them it answers, as said at each call, and never follows out of its operands."""

from __future__ import annotations

import ctypes
import math

import torch

from ..csrc.build import ensure_rounds, ensure_shared_prefix

_DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1}


def _address(t):
    return t.data_ptr() if t is not None else None


def wide_tiles_fit(head_dim: int, page_size: int, dtype) -> bool:
    """What `wide_prefix_kernel` takes."""
    return dtype == torch.bfloat16 and head_dim in (64, 128) and page_size >= 16


def wide_tiles(rows: int, kv_heads: int, shared: int, units: int) -> bool:
    """Whether the prompt's keys are multiplied in tiles of 256 columns that share them through LDS (`wide_prefix_kernel`, a launch of its
    own) rather than of 32 beside the requests' own keys.  The shared ones cost 8 to 10 us more at their start and end and less a column
    and key.  (Whole calls, narrow / wide us, 256 units, 64 own keys: 32 heads over 8 of 128, 32,768 shared, 64 rows 38 / 52, 96 49 / 51, 112
    57 / 53; 16,000 shared, 160 rows 42 / 43, 192 49 / 45, 256 57 / 49; 8,192 shared, 256 rows 35 / 42, 320 42 / 42; 2,048 shared, 960 rows
    36 / 43, 1,280 53 / 46; 16 over 4 of 64, 32,768 shared, 128 rows 24 / 29, 192 33 / 31, 256 40 / 33.  Two tiles of 32 wait
    for reads however long the prompt: 131,072 shared, 64 rows 139 / 148, 80 186 / 155.  A product of rows and keys does not know how many
    segments they make: of these points two lie on its wrong side, 32,768 shared with 96 rows (wide, 2 us more than narrow) and 2,048
    shared with 1,280 rows (narrow, 7 us more than wide).)"""
    return rows > 64 and rows * kv_heads * shared >= 85_000 * units


OWN_ROOM = 512 << 20        # bytes of own keys' partial sums


def cut_own(requests: int, rows: int, kv_heads: int, most: int, units: int, segment_bytes: int = 0) -> tuple[int, int]:
    """(segments, keys of one) of up to `most` keys that a request of up to `rows` rows a kv head holds behind the prompt.  What a block waits
    for at its start and end is a good part of its time, but a long request's keys are not to outlast the others': segments of 128 keys, a
    step for each of a block's waves, while they find a unit each, of 256 while those do, of 384 beyond, and the whole up to half as
    much again.  (8 kv heads, whole calls, us, equal lengths / up to that, segments of 128, 256, 384, 512 and about 1,000 keys: 8 requests of
    256 keys 17.3 / 16.8, 18.5 / 18.2, 20.5 / 19.7; 8 of 1,000 26 / 18, 21 / 19, 21 / 20, 22 / 22, 27 / 27; 16 of 600 25 / 18, 24 / 18,
    20 / 19, 21 / 20; 64 of 1,000 87 / 37, 66 / 32, 62 / 33, 64 / 34, 58 / 39; in a launch of their own 64 of 2,048 213 / 94, 187 / 81,
    179 / 79, 179 / 82, 179 / 89; 27 of 2,000 with up to 25 rows 145 / 68, 124 / 63, 124 / 64, 117 / 63, 111 / 67; of one segment 64 of
    500, 512 keys 39 / 30 and 384 40 / 29; with 40 rows 133 / 92 and 145 / 85.)
    The bound is the caller's, and a recorded call's the longest it may meet: a segment leaves `segment_bytes` of partial sums, as many of them as
    `OWN_ROOM` holds, but eight at least (64 requests of 5 rows, 64 heads of 128, a bound of 131,072 keys: 256 segments of 512 keys would be 2.7
    GB, 49 of 2,688 are)."""
    blocks = requests * kv_heads * ((rows + 63) // 64)
    keys = 128 if blocks * ((most + 127) // 128) <= units else 256 if blocks * ((most + 255) // 256) <= units else 384 if most > 576 else most
    segments = max(8, min(256, OWN_ROOM // segment_bytes)) if segment_bytes else 256
    keys = (max(keys, (most + segments - 1) // segments) + 127) // 128 * 128
    return (most + keys - 1) // keys, keys


def cut_prefix(columns: int, rows: int, kv_heads: int, shared: int, units: int, exact: bool) -> tuple[int, int]:
    """The same of a shared prompt, whose blocks take `columns` rows each, 256 or 32: one a unit, whatever else runs beside them - with more
    some units have two, and the others wait for those -, segments of 256 keys at least, or of 128 of less than 1,024 that are shared
    and in float32 (`exact`), whose steps take four times as long.
    (Tiles of 32 columns, 8 kv heads, whole calls, us: 32,768 shared, 48 rows, 128, 256, 320, 416 and 512 blocks 54, 35, 45, 38, 36; 96
    rows, 240, 312, 480 48, 62, 46; 8,192 shared, 64 rows, 128, 256, 352, 512 22, 18, 20, 23; 2,048 shared, 64 rows, segments of 128,
    256, 384 keys 15.7, 13.6, 14.4; of 4 kv heads 512 shared, 8 rows, 11.0, 11.5, 11.5; float32, 2,000
    shared, segments of 128 and 256 keys 16, 22.)"""
    if shared == 0:
        return 0, 32
    blocks = kv_heads * ((rows + columns - 1) // columns)
    least = 256 if shared >= 1024 and not exact else 128
    segments = max(1, min(units // blocks, (shared + least - 1) // least, 256))
    keys = ((shared + segments - 1) // segments + 127) // 128 * 128
    return (shared + keys - 1) // keys, keys


class RoundKernels:
    """Mixed into `HipKernels` (which provides `_dense`, `_check`, `_pages`, `_stream`, `device`)."""

    # a shared prompt's keys for tiles of 256 columns, whose weights are rounded once, where heads and pages allow it: None = by the sizes
    wide_prefix_tiles = None
    _rounds_lib = None

    def _rounds(self):
        if self._rounds_lib is None:
            lib = self._load(ensure_rounds())
            p, i, n = ctypes.c_void_p, ctypes.c_int, ctypes.c_long      # (with the types known, addresses are handed over as they are)
            for name, result, types in (
                    ("akv_place_most_requests", i, ()),
                    ("akv_place_tokens", i, (p, p, p, p, n, p, p, p, i, i, i, p, i, i, i, p, p, p, p, p, p, p, p, i, p)),
                    ("akv_verify_workspace", n, (i, i, i)),
                    ("akv_verify_drafts", i, (p, i, i, p, p, p, p, i, i, p, n, n, p, p, p, p))):
                getattr(lib, name).restype, getattr(lib, name).argtypes = result, types
            self._place_most = lib.akv_place_most_requests()
            self._rounds_lib = lib
        return self._rounds_lib

    def _load(self, path: str):
        try:
            return ctypes.CDLL(path)
        except OSError as error:
            raise self._error(f"the kernel library {path} could not be loaded: {error}") from error

    @staticmethod
    def _error(message: str):
        from .hip import KernelError
        return KernelError(message)

    def _shared_prefix_entry(self, head_dim: int):
        entries = self.__dict__.setdefault("_shared_prefix_entries", {})
        if head_dim not in entries:
            entry = getattr(self._load(ensure_shared_prefix(head_dim)), f"akv_attention_shared_prefix_d{head_dim}")
            p, i, n = ctypes.c_void_p, ctypes.c_int, ctypes.c_long
            entry.restype = i
            entry.argtypes = (p, p, p, p, i, p, p, p, p, p, p, p, i, i, i, n, i, i, i, n, ctypes.c_float, i, i, i, i, i, i, i, i, p)
            entries[head_dim] = entry
        return entries[head_dim]

    def _placed(self, t, name: str) -> None:
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != self.device.index:
            raise self._error(f"{name} must be a tensor on {self.device}, got {getattr(t, 'device', type(t))}")

    def _vectors(self, names, tensors, counts) -> None:
        """Checks int32 vectors.  (One loop with the comparisons in it: a call has fifteen of them and takes the device five microseconds.)"""
        index, i32 = self.device.index, torch.int32
        for t, count in zip(tensors, counts):
            if t.dtype is not i32 or t.get_device() != index or t.dim() != 1 or t.numel() != count or not t.is_contiguous():
                self._dense(t, names[[one is t for one in tensors].index(True)], i32, (count,))

    def _check_spans(self, status: int, what: str, spans) -> None:
        """`_check` of an entry that looks at what memory its operands share (csrc/common.h, `shared_spans`)."""
        if status <= -1000:
            first, second = divmod(-status - 1000, 64)
            raise self._error(f"{what}: {spans[first]} and {spans[second]} share memory")
        self._check(status, what)

    # ---- attention -----------------------------------------------------------------------------------------------------
    def attention_shared_prefix(self, q, k_pages, v_pages, block_table, q_start, seq_lens, shared, q_heads, kv_heads, head_dim, scale, out,
                                max_seq_len, max_new_tokens, rows=None, prefix_pages=None, two_part_weights=False):
        """Attention of requests whose first `shared` tokens (a multiple of the page size; 0: none) lie in the same pages: those
        are read once for all of them, so that many requests cost little more than one.  q, out [tokens, q_heads * head_dim]:
        encoded queries, request by request, whose keys and values are in the pages already.  q_start [requests + 1]: a request's
        first row; seq_lens [requests]: the tokens it holds, its new ones among them; both int32 on the device.  block_table: row r,
        or rows[r] where `rows` is given, holds request r's pages.  The prompt's are read from `prefix_pages` (its first shared / page
        size entries, as `place_tokens` takes them), or, where that is not given, from the first request's row, which must then stand
        although that request brings nothing any more.  No request holds more than `max_seq_len` tokens or brings more than
        `max_new_tokens` (0 is fine, and any number from there on; prompts of thousands of tokens are `attention`'s).
        float32 or bfloat16; head sizes as `check_attention_sizes` has them; pages of 8 tokens or more, a power of two.
        bfloat16: softmax weights are multiplied in two bfloat16 parts, the rounded one and what the rounding left, as `attention` does -
        but the weights of a prompt whose keys go in tiles of 256 columns (heads of 64 and 128, pages of 16 and more, from
        the rows and keys on that `wide_tiles` says) are rounded once, by up to 2^-8 of each: what a request gets there is off by 0.0023 of the
        output's largest in place of 0.0017, of which 0.0016 is the output's own rounding, and which of both it is depends on the batch.
        `two_part_weights`: in two parts whatever the batch, in tiles of 32 columns.
        Both bounds cost time and memory where they are far above the lengths: the launch has a block for every segment of keys that each
        request might hold, and partial sums lie in 4 * tokens * q_heads * (head_dim + 2) bytes a segment (`cut_own`, `cut_prefix`) - some
        tens of MB where bounds are tight, 600 MB at most, or eight segments of very large batches.
        A token gets NaN where its request's table (or, of the prompt, what it is read from) names a page outside the pool or is no row of
        block_table, where its request exceeds the bounds, or where it stands within the
        prompt.  Rows of `out` behind the last request's are left as they are."""
        tokens, requests = q.shape[0], seq_lens.shape[0]
        self.check_attention_sizes(q_heads, kv_heads, head_dim, 1)
        if q.dtype not in _DTYPE_CODE:
            raise self._error(f"kernels take float32 or bfloat16 tensors, got {q.dtype}")
        self._dense(q, "q", None, (tokens, q_heads * head_dim))
        self._dense(out, "out", q.dtype, (tokens, q_heads * head_dim))
        num_pages, page_size = self._pages(k_pages, v_pages, kv_heads, head_dim, q.dtype)
        if page_size < 8 or page_size & (page_size - 1):
            raise self._error(f"pages of {page_size} tokens: attention over a shared prompt takes 8 or more, a power of two")
        self._vectors(("q_start", "seq_lens"), (q_start, seq_lens), (requests + 1, requests))
        if rows is not None:
            self._dense(rows, "table rows", torch.int32, (requests,))
        if prefix_pages is not None:
            self._dense(prefix_pages, "prefix_pages", torch.int32)
            if prefix_pages.dim() != 1 or prefix_pages.shape[0] * page_size < shared:
                raise self._error(f"prefix_pages must be a vector of the pages of {shared} tokens, got {tuple(prefix_pages.shape)}")
        self._dense(block_table, "block_table", torch.int32)
        if block_table.dim() != 2 or (rows is None and block_table.shape[0] != requests):
            raise self._error(f"block_table must be [{requests if rows is None else 'rows'}, pages], got {tuple(block_table.shape)}")
        shared, max_seq_len, max_new_tokens = int(shared), int(max_seq_len), int(max_new_tokens)
        if shared < 0 or shared % page_size:
            raise self._error(f"a shared prompt of {shared} tokens is not whole pages of {page_size}")
        if max_new_tokens < 1 or max_seq_len <= shared:
            raise self._error(f"a request of up to {max_seq_len} tokens, up to {max_new_tokens} of them new, has none behind a prompt of {shared}")
        if max_seq_len > block_table.shape[1] * page_size:
            raise self._error(f"a request of {max_seq_len} tokens does not fit a block table of {block_table.shape[1]} pages")
        if not (scale > 0.0 and math.isfinite(scale)):
            raise self._error(f"the scores' scale must be positive and finite, not {scale}")
        if (q.data_ptr() | k_pages.data_ptr() | v_pages.data_ptr() | out.data_ptr()) % 16:
            raise self._error("queries, pages and the output must lie on 16-byte boundaries")
        if tokens == 0 or requests == 0:
            return
        if num_pages == 0:
            raise self._error("there are no pages")
        group = q_heads // kv_heads
        max_new_tokens, max_seq_len = min(max_new_tokens, tokens), min(max_seq_len, 2 ** 30)       # (nobody brings or holds more)
        wide = not two_part_weights and wide_tiles_fit(head_dim, page_size, q.dtype) and (
            self.wide_prefix_tiles if self.wide_prefix_tiles is not None else wide_tiles(tokens * group, kv_heads, shared, self.compute_units))
        of_segment = 4 * tokens * q_heads * (head_dim + 2)
        own_segments, own_keys = cut_own(requests, max_new_tokens * group, kv_heads, max_seq_len - shared, self.compute_units, of_segment)
        prefix_segments, prefix_keys = cut_prefix(256 if wide else 32, tokens * group, kv_heads, shared, self.compute_units, q.dtype == torch.float32)
        segments = prefix_segments + own_segments
        # (from torch's pool: a recorded call then has room of its own, and calls on other streams do not meet in one)
        room = torch.empty(segments * of_segment // 4, dtype=torch.float32, device=self.device)
        sums = room.data_ptr()
        self._check_spans(self._shared_prefix_entry(head_dim)(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), _DTYPE_CODE[q.dtype], sums,
            sums + 4 * segments * tokens * q_heads * head_dim, q_start.data_ptr(), seq_lens.data_ptr(), block_table.data_ptr(), _address(rows), _address(prefix_pages),
            block_table.shape[1], block_table.shape[0], requests, tokens, q_heads, kv_heads, page_size, num_pages, scale, shared, max_seq_len - shared, max_new_tokens,
            prefix_segments, prefix_keys, own_segments, own_keys, int(wide), self._stream()), "attention_shared_prefix",
            ("out", "q", "k_pages", "v_pages", "block_table", "q_start", "seq_lens", "table rows", "prefix_pages"))

    # ---- drafted tokens ------------------------------------------------------------------------------------------------
    def verify_drafts(self, logits, tokens, q_start, temperature, uniforms, kept, chosen, draft_logits=None):
        """How many of every request's drafted tokens the target keeps, and the token that follows them; the result is distributed as
        the target's own draws.  logits [rows, vocab] float32: the target's, for the rows q_start[r] .. q_start[r + 1] - 1 (int32) of
        request r; tokens [rows] int32: what was fed there, the request's last token and its drafts behind it.  uniforms [requests,
        places] float32 in [0, 1), places - 1 the most drafts of a request: number i for draft i, the last for the token that follows.
        temperature [requests] float32, up to 1e28 (more is taken as that); 0 (or less) keeps a draft where it is the largest logit (ties: the
        lowest id).
        draft_logits [requests, places - 1, vocab] float32: what the drafts were drawn from, at the same temperature - any strides, rows
        contiguous; None: drafts that were not drawn (looked up in a text), kept with the target's probability of them.
        kept [requests], chosen [requests, places] int32: the kept drafts, the token that follows, -1 behind it.
        A request without rows, or with rows that are not among the logits, gets 0 and -1; rows beyond `places` are not looked at.  A row
        that has no next token - a NaN, nothing above minus infinity, or (where it is drawn from) plus infinity, in the target's or the
        draft's - ends the walk with -1 as the token.  So does a number that is NaN where the walk looks at it (a draft's that it comes to, the
        last one where a token is drawn), and a temperature that is NaN at its first row.  A draft that is no id of the vocabulary is not kept."""
        if logits.dim() != 2 or uniforms.dim() != 2:
            raise self._error("logits and uniforms must be matrices")
        (count, vocab), (requests, places) = logits.shape, uniforms.shape
        self._dense(logits, "logits", torch.float32)
        self._vectors(("tokens", "q_start", "kept"), (tokens, q_start, kept), (count, requests + 1, requests))
        self._dense(temperature, "temperature", torch.float32, (requests,))
        self._dense(uniforms, "uniforms", torch.float32)
        self._dense(chosen, "chosen", torch.int32, (requests, places))
        strides = (0, 0)
        if draft_logits is not None and places > 1:
            self._placed(draft_logits, "draft_logits")
            if draft_logits.dtype != torch.float32 or draft_logits.shape != (requests, places - 1, vocab):
                raise self._error(f"draft_logits must be float32 [{requests}, {places - 1}, {vocab}], got {draft_logits.dtype} {tuple(draft_logits.shape)}")
            if vocab > 1 and draft_logits.stride(2) != 1:
                raise self._error("draft_logits must have contiguous rows")
            strides = draft_logits.stride()[:2]
        elif draft_logits is not None:
            draft_logits = None
        if requests == 0:
            return
        lib = self._rounds()
        room = lib.akv_verify_workspace(requests, places, vocab)
        if room < 0:
            raise self._error(f"verify_drafts: {requests} requests of up to {places} rows of {vocab} logits: at most 65,535, 64 and 262,144 are taken")
        workspace = torch.empty(room, dtype=torch.uint8, device=self.device)
        self._check_spans(lib.akv_verify_drafts(
            logits.data_ptr(), count, vocab, tokens.data_ptr(), q_start.data_ptr(), temperature.data_ptr(), uniforms.data_ptr(), requests, places,
            _address(draft_logits), strides[0], strides[1], kept.data_ptr(), chosen.data_ptr(), workspace.data_ptr(), self._stream()),
            "verify_drafts", ("kept", "chosen", "logits", "tokens", "q_start", "temperature", "uniforms", "draft_logits"))

    _PLACED = ("lengths", "counts", "held", "free_pages", "cursor", "q_start", "seq_lens", "held_after", "cursor_after", "positions", "seq_of_token",
               "slot_map", "status")

    # ---- a step's layout -----------------------------------------------------------------------------------------------
    def place_tokens(self, lengths, counts, held, free_pages, cursor, table, page_size, q_start, seq_lens, held_after, cursor_after, positions,
                     seq_of_token, slot_map, status, rows=None, prefix_pages=None, clear_rest=False):
        """A step's layout from lengths on the device (all int32).  lengths, counts, held [requests]: the tokens a request holds, those it
        brings, and its pages.  It takes the pages it lacks from free_pages[cursor ...], in the requests' order; they are entered into its
        row of `table` (row r, or rows[r]), and held_after [requests] and cursor_after [1] say what is held and taken then.  A request
        that holds no page starts on `prefix_pages`, if they are given: they are entered too, and `lengths` counts their tokens.  What it
        brings at places within them is written into them: so a prompt is filled, by a batch none of whose requests has it yet, a place
        by one request at most - other batches are refused (-4), those outside the batch nobody sees.  (Where some requests of a batch start on
        the prompt and others without one, the caller enters its pages into the rows of the former, counts them in `held`, and gives no
        prefix_pages.)
        q_start [requests + 1], seq_lens [requests] (the tokens held after the step); positions, seq_of_token and slot_map [tokens]: of
        every token, request by request; tokens are all that the requests bring, or more: entries behind the last are left as they are.  A
        token whose page is negative, or so far that its slot does not fit 31 bits, has slot -1.
        status [1]: the pages taken, or, with nothing else written, -1 too few free pages, -2 a row that the table does not have, that is too
        narrow or that two requests name, -3 more tokens than the maps have room for, -4 a negative number, fewer pages than a length
        fills, or a request that brings places of the prompt's pages beside one that has pages, starts behind the prompt or brings the same
        places.
        What is left as it is names the layout before: a cache write over the whole of `slot_map` would follow it.  `clear_rest`, for rounds in
        which no host looks at counts and status: slot_map is -1 behind the last token (`kv_write` leaves such rows alone), and where the step
        cannot be laid out nobody brings anything - slot_map all -1, q_start all 0, seq_lens the lengths, held_after and cursor_after as
        held and cursor are -, so that attention writes nothing and `verify_drafts` answers 0 kept and -1."""
        requests, tokens = lengths.shape[0], positions.shape[0]
        lib = self._rounds()
        free = free_pages.shape[0]
        self._vectors(self._PLACED, (lengths, counts, held, free_pages, cursor, q_start, seq_lens, held_after, cursor_after, positions, seq_of_token,
                                     slot_map, status),
                      (requests, requests, requests, free, 1, requests + 1, requests, requests, 1, tokens, tokens, tokens, 1))
        if rows is not None:
            self._dense(rows, "table rows", torch.int32, (requests,))
        if prefix_pages is not None:
            self._dense(prefix_pages, "prefix_pages", torch.int32, (prefix_pages.shape[0],))
        self._dense(table, "table", torch.int32)
        if table.dim() != 2 or (rows is None and table.shape[0] < requests):
            raise self._error(f"table must be a matrix with a row for each of {requests} requests, got {tuple(table.shape)}")
        if page_size < 1 or page_size != int(page_size):
            raise self._error(f"page_size {page_size} must be a positive number of tokens")
        if requests > self._place_most:
            raise self._error(f"{requests} requests in one step; at most {self._place_most} are taken")
        self._check_spans(lib.akv_place_tokens(
            lengths.data_ptr(), counts.data_ptr(), held.data_ptr(), free_pages.data_ptr(), free, cursor.data_ptr(),
            table.data_ptr(), _address(rows), table.shape[0], table.shape[1], int(page_size), _address(prefix_pages),
            prefix_pages.shape[0] if prefix_pages is not None else 0, requests, tokens, q_start.data_ptr(), seq_lens.data_ptr(),
            held_after.data_ptr(), cursor_after.data_ptr(), positions.data_ptr(), seq_of_token.data_ptr(), slot_map.data_ptr(),
            status.data_ptr(), int(bool(clear_rest)), self._stream()), "place_tokens",
            ("q_start", "seq_lens", "held_after", "cursor_after", "positions", "seq_of_token", "slot_map", "status", "table", "lengths", "counts",
             "held", "cursor", "free_pages", "table rows", "prefix_pages"))
