"""A paged KV cache held in 4 bits, with the attention that reads it (``vuib_kv4_*`` of libvuib200).

Next to the engine's bf16 cache of ``max_seq`` positions a slot (48 KB a position for Vui Nano), for servers that keep
many or long conversations: positions live in blocks that any sequence may own, and keys and values take 5 bits an
element with their scales (3.2 times less memory, and 3.2 times fewer bytes for a decode step to read).  The block
tables are built and extended on the GPU, so that a captured step needs no host when a sequence crosses into a new
block.  The reference has no counterpart.

A step::

    plan = cache.plan(slots)                       # one new row for every sequence: tables, positions, slot map
    for layer in range(n_layers):
        cache.append(layer, k, v, plan)            # (rows, n_kv_heads, head_dim) bf16, keys with RoPE applied
        out = cache.attention(layer, q, plan)      # (rows, n_heads, head_dim) bf16

A prompt is the same with ``cache.plan(slots, lengths)``; its rows are the sequences' new positions behind one another.
"""

from __future__ import annotations

import contextlib
import ctypes as C

import torch
from torch import Tensor

from . import _lib

_NOTHING = contextlib.nullcontext()
# the current stream's handle; torch's public call builds a stream object first (2 us of a call that takes 15)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


_MOST_ROWS = 1 << 24      # of a plan


def _int32(x: int) -> int:
    """x, or the end of 32 bits that is next to it: out of range all the same, where ctypes would drop the higher bits."""
    return min(max(x, -2 ** 31), 2 ** 31 - 1)


class Kv4Plan:
    """The rows of one step, all on the device: ``row_slot`` and ``row_pos`` (int32) say which position of which sequence
    a row is, ``slot_map`` (int64) where it lies (block * block_size + offset), ``cu_rows`` (int32, one more than
    sequences) where each sequence's rows begin.  Rows behind the last are -1.  The calls that take a plan read these
    arrays, those in a captured graph at every replay: the plan has to live as long."""

    def __init__(self, cache: "Kv4Cache", n_seqs: int, n_rows: int, max_new: int):
        device, self._cache = cache.device, cache
        self.n_seqs, self.n_rows, self.max_new = n_seqs, n_rows, max_new
        work = (7 * n_seqs + 3 + n_rows + 3) & ~3          # the parts behind it: 16-byte aligned
        row = (n_rows + 3) & ~3
        # one allocation: work, slot_map (int64), row_slot, row_pos, cu_rows
        self._ints = torch.empty(work + 4 * row + n_seqs + 1, dtype=torch.int32, device=device)
        self._at = (work, work + 2 * row, work + 3 * row, work + 4 * row)
        at = self._ints.data_ptr()
        self._c = _lib.VuibKv4Plan(n_seqs, n_rows, max_new, at, at + 4 * self._at[3], at + 4 * self._at[1], at + 4 * self._at[2], at + 4 * work)
        self._ref = C.byref(self._c)
        self._ws_bytes = -1        # of its attention calls, asked for once
        self._ws: dict[int, Tensor] = {}      # by stream

    @property
    def slot_map(self) -> Tensor:
        return self._ints[self._at[0]:self._at[0] + 2 * self.n_rows].view(torch.int64)

    @property
    def row_slot(self) -> Tensor:
        return self._ints[self._at[1]:self._at[1] + self.n_rows]

    @property
    def row_pos(self) -> Tensor:
        return self._ints[self._at[2]:self._at[2] + self.n_rows]

    @property
    def cu_rows(self) -> Tensor:
        return self._ints[self._at[3]:]


class Kv4Cache:
    """``n_blocks`` blocks of ``block_size`` positions (16, 32, 64, 128 or 256) for ``max_seqs`` sequences of at most
    ``max_blocks`` blocks each; ``head_dim`` 64, 96 or 128, up to 16 query heads per kv head.  ``seq_lens``,
    ``block_table`` and ``n_free`` are the device's own state, to be read but not written by the caller."""

    def __init__(self, *, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int, n_blocks: int, block_size: int = 64,
                 max_seqs: int, max_blocks: int | None = None, device="cuda"):
        self._h = C.c_void_p()
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError(f"device {dev}: a CUDA device is wanted; there is no CPU path")
        max_blocks = n_blocks if max_blocks is None else max_blocks
        sizes = (n_layers, n_heads, n_kv_heads, head_dim, n_blocks, block_size, max_seqs, max_blocks)
        cfg = _lib.VuibKv4Config(*(_int32(x) for x in sizes))
        self._lib = _lib.load()
        rc = self._lib.vuib_kv4_create(C.byref(cfg), C.byref(self._h))
        if rc:
            raise ValueError(f"unsupported 4-bit cache (status {rc}): {n_layers} layers, {n_heads}/{n_kv_heads} heads of {head_dim}, "
                             f"{n_blocks} blocks of {block_size}, {max_seqs} sequences of up to {max_blocks} blocks")
        if not torch.cuda.is_available():
            raise RuntimeError("vui_b200.Kv4Cache needs a CUDA device (sm_100a); there is no CPU path")
        self.device = dev if dev.index is not None else torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index
        self.n_layers, self.n_heads, self.n_kv_heads, self.head_dim = n_layers, n_heads, n_kv_heads, head_dim
        self.n_blocks, self.block_size, self.max_seqs, self.max_blocks = n_blocks, block_size, max_seqs, max_blocks
        n = C.c_size_t()
        self._ck(self._lib.vuib_kv4_pool_bytes(self._h, C.byref(n)))
        self.pool_bytes = n.value
        i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=self.device)  # noqa: E731
        with self._here():
            self._pool = torch.zeros(n.value, dtype=torch.uint8, device=self.device)
            self.seq_lens, self.block_table = i32(max_seqs), i32(max_seqs, max_blocks)
            self._free, self.n_free, self._flag = i32(n_blocks), i32(1), i32(1)
            P = lambda t: t.data_ptr()  # noqa: E731
            self._ck(self._lib.vuib_kv4_bind(self._h, P(self._pool), n.value, P(self.seq_lens), P(self.block_table), P(self._free),
                                             P(self.n_free), P(self._flag)))
            self._ck(self._lib.vuib_kv4_reset(self._h, self._stream))

    def __del__(self):
        try:
            if self._h:
                self._lib.vuib_kv4_destroy(self._h)
                self._h = C.c_void_p()
        except Exception:
            pass

    def _ck(self, rc: int) -> None:
        if rc:
            buf = C.create_string_buffer(256)
            self._lib.vuib_kv4_last_error(self._h, buf, 256)
            raise _lib.VuibError(rc, buf.value.decode(errors="replace") or "(no message)")

    @property
    def _stream(self):
        return _raw_stream(self._index)

    def _here(self):
        """Makes the cache's device the current one, where it is not."""
        return _NOTHING if torch.cuda.current_device() == self._index else torch.cuda.device(self._index)

    def _ints(self, v, name: str, n: int | None = None) -> Tensor:
        t = v if torch.is_tensor(v) else torch.as_tensor(v, dtype=torch.int64 if len(v) == 0 else None)
        if t.dtype is torch.int32 and t.device == self.device and t.dim() == 1 and t.is_contiguous() and (n is None or t.numel() == n):
            return t
        if t.dim() != 1 or t.is_floating_point() or t.is_complex() or (n is not None and t.numel() != n):
            raise ValueError(f"{name}: a one-dimensional list of {'whole numbers' if n is None else f'{n} whole numbers'} is wanted, "
                             f"got {t.dtype} {tuple(t.shape)}")
        if t.dtype is torch.uint64:
            raise ValueError(f"{name}: int32 or int64 is wanted, got {t.dtype}")
        if t.dtype in (torch.uint16, torch.uint32):
            t = t.to(torch.int64)
        if not t.is_cuda and t.numel() and not (-2 ** 31 <= int(t.min()) and int(t.max()) < 2 ** 31):
            raise ValueError(f"{name}: numbers beyond 32 bits")
        if t.is_cuda and t.dtype is torch.int64:      # the ends of 32 bits, which are out of range too
            t = t.clamp(-2 ** 31, 2 ** 31 - 1)
        return t.to(self.device, torch.int32).contiguous()

    # ------------------------------------------------------------------ tables
    def reset(self) -> None:
        """Empties every sequence."""
        with self._here():
            self._ck(self._lib.vuib_kv4_reset(self._h, self._stream))

    def plan(self, slots, new_lens=None, at=None, *, n_rows: int | None = None, max_new: int | None = None) -> Kv4Plan:
        """Lengthens sequence ``slots[i]`` by ``new_lens[i]`` positions (None: one each), after cutting it back to ``at[i]``
        where ``at`` is given, and lays out the new rows.  Lists or tensors; with lengths that are on the device, ``n_rows``
        (rows that the plan has room for) and ``max_new`` (most rows of one sequence) have to be given, so that nothing waits
        for them.  Slot -1 takes no part.  A sequence for which rows or blocks run out, or whose numbers are out of range,
        stays as it is, brings no rows and is recorded (``check_device``)."""
        if new_lens is not None and not (torch.is_tensor(new_lens) and new_lens.is_cuda):
            host = [int(x) for x in new_lens]
            n_rows = sum(max(x, 0) for x in host) if n_rows is None else n_rows
            max_new = min(n_rows, max(host, default=0)) if max_new is None else max_new
        slots = self._ints(slots, "slots")
        n = slots.numel()
        if n == 0:
            raise ValueError("slots is empty")
        if new_lens is None:
            n_rows, max_new = n if n_rows is None else n_rows, 1 if max_new is None else max_new
        if n_rows is None or max_new is None:
            raise ValueError("new_lens on the device need n_rows and max_new")
        with self._here():
            new = None if new_lens is None else self._ints(new_lens, "new_lens", n)
            at = None if at is None else self._ints(at, "at", n)
            if n_rows < 0 or max_new < 0:
                raise ValueError("n_rows and max_new must not be negative")
            if n_rows > _MOST_ROWS:
                raise ValueError(f"n_rows {n_rows}: a plan holds up to {_MOST_ROWS}")
            plan = Kv4Plan(self, n, int(n_rows), min(int(max_new), int(n_rows)))
            self._ck(self._lib.vuib_kv4_plan(self._h, plan._ref, slots.data_ptr(), None if new is None else new.data_ptr(),
                                             None if at is None else at.data_ptr(), self._stream))
        return plan

    def release(self, slots) -> None:
        """Empties these sequences and gives their blocks back."""
        slots = self._ints(slots, "slots")
        none = torch.zeros_like(slots)
        self.plan(slots, none, at=none, n_rows=0, max_new=0)

    # -------------------------------------------------------------------- rows
    def _own(self, plan: Kv4Plan) -> None:
        if not isinstance(plan, Kv4Plan) or plan._cache is not self:
            raise ValueError("plan: one that this cache made is wanted")

    def _rows(self, t: Tensor, name: str, n: int, heads: int, *, out: bool = False) -> Tensor:
        """(n, heads, head_dim) or (n, heads * head_dim) as the library takes it: bf16 on this device, heads behind one
        another, rows a multiple of 16 bytes apart.  An input that lies otherwise, or is of another type or device, is copied (and
        rounded to bf16), an output refused."""
        if torch.is_tensor(t) and t.dtype is torch.bfloat16 and t.device == self.device and t.shape == (n, heads, self.head_dim) and \
                t.is_contiguous() and t.data_ptr() % 16 == 0:
            return t
        if not torch.is_tensor(t) or tuple(t.shape) not in ((n, heads, self.head_dim), (n, heads * self.head_dim)):
            raise ValueError(f"{name}: ({n}, {heads}, {self.head_dim}) is wanted, got {tuple(t.shape) if torch.is_tensor(t) else type(t)}")
        good = t.device == self.device and t.dtype == torch.bfloat16
        if not out:
            t = t.to(self.device, torch.bfloat16)
        flat = t.stride(-1) == 1 and (t.dim() == 2 or heads == 1 or t.stride(1) == self.head_dim)
        step = t.stride(0) if n > 1 else heads * self.head_dim
        if flat and step % 8 == 0 and step >= heads * self.head_dim and t.data_ptr() % 16 == 0 and (good or not out):
            return t
        if out:
            raise ValueError(f"{name}: bf16 on {self.device} with heads behind one another and rows a multiple of 16 bytes apart is wanted")
        t = t.contiguous()
        return t if t.data_ptr() % 16 == 0 else t.clone()

    def _step(self, t: Tensor, heads: int) -> int:
        return t.stride(0) if t.shape[0] > 1 else heads * self.head_dim

    def append(self, layer: int, k: Tensor, v: Tensor, plan: Kv4Plan) -> None:
        """Stores the plan's rows: k, v (n_rows, n_kv_heads, head_dim), keys with RoPE applied.  NaN is stored as 0 and
        magnitudes beyond 60000 as 60000, which ``check_device`` reports.  Other types than bf16, other devices and rows that are not
        16-byte aligned are copied first."""
        self._own(plan)
        with self._here():
            n, heads = plan.n_rows, self.n_kv_heads
            k, v = self._rows(k, "k", n, heads), self._rows(v, "v", n, heads)
            rc = self._lib.vuib_kv4_append(self._h, _int32(layer), plan._ref, k.data_ptr(), self._step(k, heads), v.data_ptr(), self._step(v, heads),
                                           _raw_stream(self._index))
            if rc:
                self._ck(rc)

    def read(self, layer: int, row_slot, row_pos, *, k_out: Tensor | None = None, v_out: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """The keys and values stored for position ``row_pos[i]`` of sequence ``row_slot[i]``: (n, n_kv_heads, head_dim) bf16,
        new tensors or ``k_out`` and ``v_out`` (a stretch of an engine's bf16 cache, say).  Slot -1 gives zeros; so do positions that
        the sequence does not have, which are recorded (``check_device``)."""
        with self._here():
            row_slot = self._ints(row_slot, "row_slot")
            n = row_slot.numel()
            row_pos = self._ints(row_pos, "row_pos", n)
            new = lambda: torch.empty(n, self.n_kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.device)  # noqa: E731
            k = new() if k_out is None else self._rows(k_out, "k_out", n, self.n_kv_heads, out=True)
            v = new() if v_out is None else self._rows(v_out, "v_out", n, self.n_kv_heads, out=True)
            if n:
                self._ck(self._lib.vuib_kv4_read(self._h, _int32(layer), n, row_slot.data_ptr(), row_pos.data_ptr(), k.data_ptr(),
                                                 self._step(k, self.n_kv_heads), v.data_ptr(), self._step(v, self.n_kv_heads), self._stream))
        return k, v

    def attention(self, layer: int, q: Tensor, plan: Kv4Plan, *, scale: float | None = None, out: Tensor | None = None) -> Tensor:
        """Causal attention of the plan's rows, each over its sequence up to and with its own position (append first):
        q (n_rows, n_heads, head_dim) with RoPE applied -> the same shape, bf16.  ``scale`` defaults to 1 / sqrt(head_dim).
        Rows behind the plan's last are not written.  ``q`` is copied first where ``append`` would copy.

        All of a plan's rows are served in one way, by its ``max_new``: a prompt's chunk of a hundred rows and more and single tokens of
        other sequences in one step are faster as two plans, and the single tokens then have the bits of a step of their own."""
        if scale is not None and not (scale <= 1e30 and C.c_float(scale).value > 0):       # 0 is the library's word for the default
            raise ValueError("scale must be positive, also in 32 bits, and at most 1e30")
        self._own(plan)
        if torch.cuda.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.attention(layer, q, plan, scale=scale, out=out)
        rows, heads, width = plan.n_rows, self.n_heads, self.n_heads * self.head_dim
        q = self._rows(q, "q", rows, heads)
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=self.device)
            step = width
        else:
            out = self._rows(out, "out", rows, heads, out=True)
            step = self._step(out, heads)
        stream = _raw_stream(self._index)
        if plan._ws_bytes < 0:
            n = C.c_size_t()
            self._ck(self._lib.vuib_kv4_attention_workspace(self._h, plan._ref, C.byref(n)))
            plan._ws_bytes = n.value
        ws = None
        if plan._ws_bytes:
            # calls on one stream follow one another and share the plan's workspace; a captured call has its own, which its graph keeps
            ws = plan._ws.get(stream)
            if ws is None or torch.cuda.is_current_stream_capturing():
                ws = torch.empty(plan._ws_bytes, dtype=torch.uint8, device=self.device)
                if not torch.cuda.is_current_stream_capturing():
                    plan._ws[stream] = ws
        rc = self._lib.vuib_kv4_attention(self._h, _int32(layer), plan._ref, q.data_ptr(), self._step(q, heads), out.data_ptr(), step, scale or 0.0,
                                          None if ws is None else ws.data_ptr(), plan._ws_bytes, stream)
        if rc:
            self._ck(rc)
        return out

    # ------------------------------------------------------------- diagnostics
    def check_device(self) -> None:
        """Raises if a call since the last check met a slot, length or value out of range, or ran out of rows or blocks."""
        with self._here():
            self._ck(self._lib.vuib_kv4_check_flag(self._h, self._stream))

    def launch_count(self) -> int:
        return int(self._lib.vuib_kv4_launch_count(self._h))
