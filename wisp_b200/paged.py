"""A paged key/value cache for a batch of sequences, and the operators that work on it.

* ``rope_append``       rotary positions on q and k, k and v appended to the cache's pages
* ``attention``         causal attention over the pages: prompts, chunks and single tokens,
  with a sliding window and a few first tokens (sinks) that stay visible
* ``prefix_attention``  the same for sequences that share a long prefix (read once per group)
* ``copy_pages``        pages copied inside the pool of all layers
* ``PagePool``          the host-side owner of page numbers: open, extend, fork (copy on
  write), truncate, close, compact
* ``rope_frequencies``  rotary frequencies, plain or stretched for a long context

Pages are ``[n_pages, page_size, n_kv_heads, head_dim]`` per layer (``[n_layers, ...]`` for
the page operators), fp16 or bf16, one tensor for the keys and one for the values.  Every call
runs on the caller's current CUDA stream and synchronises nothing; lengths and page tables are
device tensors, so a captured step can be replayed after they changed.  torch is used for
device memory and streams only; every kernel is in ``libwisp_b200.so``.
"""

from __future__ import annotations

import ctypes as C
import importlib.util
import math

import torch

from .lib import LIB_PATH, WispErrCtx, WispError, check, lib

_binding = None


def _fail(code: int, message: str, file: bytes, line: int) -> None:
    err = WispErrCtx(code, message.encode(), file or None, line)
    raise WispError(err, code)


def _torch():
    """The binding module (raises if it has not been built)."""
    global _binding
    if _binding is None:
        path = LIB_PATH.parent / "_paged_torch.so"
        if not path.exists():
            raise ImportError(f"{path} is missing: run `python -m wisp_b200.build`")
        spec = importlib.util.spec_from_file_location("_paged_torch", path)
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        L = lib()
        m.init(*(C.cast(f, C.c_void_p).value for f in
                 (L.wisp_paged_attention_workspace_bytes, L.wisp_paged_attention,
                  L.wisp_prefix_attention, L.wisp_rope_append, L.wisp_pages_copy)), _fail)
        _binding = m
    return _binding


class TokenBatch:
    """The tokens of one step, sequence after sequence (``WispTokenBatch``).

    ``q_start`` int32 ``[n_seq + 1]``: first token of each sequence; ``kv_len`` int32
    ``[n_seq]``: cached positions, the step's own tokens included; ``table`` int32
    ``[n_seq, pages]``: the sequences' page numbers; ``max_q``: no sequence has more tokens.
    One batch serves every layer of a step."""

    __slots__ = ("q_start", "kv_len", "table", "max_q")

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, table: torch.Tensor,
                 max_q: int):
        (_binding or _torch()).check_batch(q_start, kv_len, table, max_q)
        self.q_start, self.kv_len, self.table, self.max_q = q_start, kv_len, table, max_q


def rope_frequencies(dim: int, theta: float = 10000.0, *, scaling: str | None = None,
                     factor: float = 1.0, original: int = 4096, low: float = 1.0,
                     high: float = 32.0, device=None) -> tuple[torch.Tensor, float]:
    """(inverse frequencies ``[dim // 2]`` in float64, gain) of a rotary window of ``dim``.

    ``scaling``: None; ``"linear"`` (every frequency / factor); ``"base"`` (theta raised so
    that the slowest pair is stretched by factor and the fastest kept); ``"by_parts"``: pairs
    that make fewer than ``low`` turns in ``original`` positions are divided by factor, those of
    more than ``high`` kept, those between blended in proportion to their turns, and the rows
    scaled by ``0.1 ln(factor) + 1``.  Models were also trained with blends that are linear in the
    pair's index, with other bounds or without the gain: give the operators frequencies and a gain
    of your own for those."""
    if dim <= 0 or dim % 2 or factor < 1.0 or theta <= 0:
        raise ValueError(f"rope_frequencies: dim {dim} (even), theta {theta}, factor {factor} (>= 1)")
    i = torch.arange(dim // 2, dtype=torch.float64)
    gain = 1.0
    if scaling == "base":
        theta = theta * factor ** (dim / (dim - 2)) if dim > 2 else theta
    f = theta ** (-2.0 * i / dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_parts":
        if not 0 <= low < high or original <= 0:
            raise ValueError(f"rope_frequencies: turns {low} to {high} in {original} positions")
        keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"rope_frequencies: unknown scaling {scaling!r}")
    return f.to(device) if device is not None else f, gain


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
                v_pages: torch.Tensor, batch: TokenBatch, inv_freq: torch.Tensor, *,
                q_out: torch.Tensor | None = None, offset: int = 0, interleaved: bool = False,
                gain: float = 1.0, positions: torch.Tensor | None = None,
                status: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q ``[T, heads, dim]`` and k ``[T, kv_heads, dim]`` of the batch's tokens, store k
    and v at the tokens' positions of the pages; returns the rotated q (``q_out``, by default a
    new tensor of q's dtype; ``q`` itself is allowed).

    The window of ``2 * len(inv_freq)`` dims at ``offset`` of each head is turned: pairs are
    (i, i + half) or, ``interleaved``, neighbours.  ``inv_freq`` float64 on the device
    (``rope_frequencies``); ``positions`` int32 ``[T]`` replaces the cache positions in the
    angle.  ``status``: an int32 word that gets bit 0 set for a page number outside the pool."""
    return (_binding or _torch()).rope_append(
        q, k, v, k_pages, v_pages, batch, inv_freq, q_out, offset, interleaved, gain, positions,
        status)


def attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, batch: TokenBatch, *,
              out: torch.Tensor | None = None, scale: float | None = None, window: int = 0,
              sinks: int = 0, return_lse: bool = False, workspace: torch.Tensor | None = None,
              status: torch.Tensor | None = None):
    """Causal attention of the batch's tokens over their sequences' cached positions.

    q ``[T, heads, dim]`` in fp32 or the pages' dtype; the result has q's dtype.  ``window`` > 0:
    token i sees position j when i - j < window or j < ``sinks``.  ``scale`` defaults to
    dim ** -0.5.  ``return_lse``: also the rows' log-sum-exp, fp32 ``[T, heads]`` (-inf for a row
    that sees nothing; its result is zero).  ``workspace``: uint8, at least
    ``workspace_bytes``; by default taken from torch's allocator for the call.  ``out`` must not
    overlap q.  ``status``: an int32 word that gets the bits of ``paged.status`` OR-ed in; without it
    (and without a workspace to ask) a bad page, a cut length or a wait that ran out stays unseen."""
    return (_binding or _torch()).attend(
        q, k_pages, v_pages, batch, None, None, out, scale, window, sinks, return_lse, workspace,
        status)


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     batch: TokenBatch, groups: torch.Tensor, prefix_len: torch.Tensor, *,
                     out: torch.Tensor | None = None, scale: float | None = None, window: int = 0,
                     sinks: int = 0, return_lse: bool = False,
                     workspace: torch.Tensor | None = None,
                     status: torch.Tensor | None = None):
    """``attention`` for sequences that share prefixes: the sequences ``groups[g]`` to
    ``groups[g + 1]`` hold their first ``prefix_len[g]`` positions in the same pages, which are
    read once for all of the group.  Both int32 on the device."""
    return (_binding or _torch()).attend(
        q, k_pages, v_pages, batch, groups, prefix_len, out, scale, window, sinks, return_lse,
        workspace, status)


def workspace_bytes(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    batch: TokenBatch, n_groups: int = 0) -> int:
    """Bytes of workspace an ``attention`` (or, with groups, ``prefix_attention``) call takes."""
    return (_binding or _torch()).workspace_bytes(q, k_pages, v_pages, batch, n_groups)


def status(workspace: torch.Tensor) -> int:
    """The status word of the last attention call on ``workspace`` (0: nothing wrong; bit 0: a
    page number outside the pool; bit 1: a length beyond the page table; bit 3: a wait ran out).
    Synchronises the current stream."""
    return int(lib().wisp_moe_status(workspace.data_ptr(),
                                     torch.cuda.current_stream(workspace.device).cuda_stream))


def wait_limit(seconds: float) -> float:
    """How long a wait inside an attention kernel may take (2 s at first) before the call gives up
    with bit 3 of its status; for the calls made from now on.  Returns the limit before."""
    if not 0 <= seconds < 1e9:
        raise ValueError(f"wait_limit: {seconds} seconds")
    return lib().wisp_paged_wait_limit(int(seconds * 1e9)) / 1e9


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src, dst) -> None:
    """Copy pages ``src[i]`` to ``dst[i]`` (host integers) in every layer of pools
    ``[n_layers, n_pages, page_size, n_kv_heads, head_dim]`` (or one layer's four dimensions).
    No page may be both a source and a destination, or twice a destination."""
    (_binding or _torch()).copy_pages(k_pages, v_pages, src, dst)


class PagePool:
    """Which sequence holds which pages of a pool (``wisp_page_pool_*``); host side only.

    ``extend`` gives a sequence room and replaces a shared page that is about to be written by
    one of its own; ``fork`` shares all pages of a sequence with a new one; ``compact`` renumbers
    the pages in use to the lowest numbers.  The page copies that these need are queued:
    ``apply`` runs them on the pools of all layers, and must be called before the pages are
    next written or read."""

    def __init__(self, n_pages: int, page_size: int):
        err = WispErrCtx()
        self.n_pages, self.page_size = n_pages, page_size
        self._h = lib().wisp_page_pool_create(n_pages, page_size, C.byref(err))
        if not self._h:
            raise WispError(err)
        self._destroy = lib().wisp_page_pool_destroy  # (`lib` may be gone when the pool goes)

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            self._destroy(h)

    def _id(self, rc: int, err: WispErrCtx) -> int:
        if rc < 0:
            raise WispError(err)
        return rc

    @property
    def free_pages(self) -> int:
        return lib().wisp_page_pool_free_pages(self._h)

    def open(self) -> int:
        err = WispErrCtx()
        return self._id(lib().wisp_page_pool_open(self._h, C.byref(err)), err)

    def extend(self, seq: int, length: int) -> None:
        err = WispErrCtx()
        check(lib().wisp_page_pool_extend(self._h, seq, length, C.byref(err)), err)

    def truncate(self, seq: int, length: int) -> None:
        err = WispErrCtx()
        check(lib().wisp_page_pool_truncate(self._h, seq, length, C.byref(err)), err)

    def fork(self, seq: int) -> int:
        err = WispErrCtx()
        return self._id(lib().wisp_page_pool_fork(self._h, seq, C.byref(err)), err)

    def close(self, seq: int) -> None:
        err = WispErrCtx()
        check(lib().wisp_page_pool_close(self._h, seq, C.byref(err)), err)

    def compact(self) -> int:
        err = WispErrCtx()
        return self._id(lib().wisp_page_pool_compact(self._h, C.byref(err)), err)

    def length(self, seq: int) -> int:
        err = WispErrCtx()
        return self._id(lib().wisp_page_pool_length(self._h, seq, C.byref(err)), err)

    def pages(self, seq: int) -> list[int]:
        err = WispErrCtx()
        n = self._id(lib().wisp_page_pool_pages(self._h, seq, None, 0, C.byref(err)), err)
        buf = (C.c_int * max(1, n))()
        self._id(lib().wisp_page_pool_pages(self._h, seq, buf, n, C.byref(err)), err)
        return list(buf[:n])

    def moves(self) -> tuple[list[int], list[int]]:
        """Drain the queued moves: (sources, destinations)."""
        src, dst = (C.c_int * self.n_pages)(), (C.c_int * self.n_pages)()
        s: list[int] = []
        d: list[int] = []
        while n := lib().wisp_page_pool_moves(self._h, src, dst, self.n_pages):
            s += src[:n]
            d += dst[:n]
        return s, d

    def apply(self, k_pages: torch.Tensor, v_pages: torch.Tensor) -> int:
        """Run the queued moves on the pools of all layers; how many there were.  What a refused
        copy leaves undone stays queued, for another call."""
        n = lib().wisp_page_pool_queued(self._h, None, None, 0)
        src, dst = (C.c_int * n)(), (C.c_int * n)()
        lib().wisp_page_pool_queued(self._h, src, dst, n)
        s, d = src[:n], dst[:n]
        at, touched, written = 0, set(), set()
        for i in range(n + 1):
            # (a destination met before: the page was freed and taken again in between)
            if i == n or d[i] in touched or s[i] in written:
                if i > at:
                    copy_pages(k_pages, v_pages, s[at:i], d[at:i])
                    lib().wisp_page_pool_moves(self._h, src, dst, i - at)
                at, touched, written = i, set(), set()
            if i < n:
                touched |= {s[i], d[i]}
                written.add(d[i])
        return n

    def table(self, seqs, width: int | None = None, device=None) -> torch.Tensor:
        """The sequences' page numbers, int32 ``[len(seqs), width]`` (0 where a row is shorter)."""
        rows = [self.pages(s) if s is not None else [] for s in seqs]
        w = max([1] + [len(r) for r in rows]) if width is None else width
        if any(len(r) > w for r in rows):
            raise ValueError(f"table: a sequence has more than {w} pages")
        t = torch.tensor([r + [0] * (w - len(r)) for r in rows], dtype=torch.int32).view(-1, w)
        return t.to(device) if device is not None else t
