"""A batch of sequences through a decoder stack: the paged cache's operators around the MoE block.

``BatchDecoder`` is the batched form of the engine's one-sequence decoder step (GQA / MHA
attention, MoE feed-forward): each ``step`` takes new tokens of any number of sequences (a
prompt, a chunk, a single token each, in one batch) through

    x = embed[token]
    per layer:  q, k, v = projections of rmsnorm(x);  rotary positions, k and v to the pages
                x += o_proj(attention over the pages)
                x += MoE(rmsnorm(x))
    logits = lm_head . rmsnorm(x) of each sequence's last token

Sequences share pages: ``fork`` continues one sequence in several ways, and a step whose
neighbouring sequences begin with the same pages reads those once (``prefix_attention``).  The
projections are plain fp16 matrix products; everything else runs in this library's kernels.

The one-sequence step keeps 32 bits everywhere but in the cache.  Here the inputs of the matrix
products are rounded to fp16, the weights' type, so that they run on the tensor cores; their sums,
the residual and the logits are fp32.  q, k, v and the attention rows are fp16 by default, which is
what prompts are fast in; ``rows=torch.float32`` keeps them in fp32.
"""

from __future__ import annotations

from contextlib import suppress
from dataclasses import dataclass
from operator import index

import torch

from . import paged
from .moe import MoEStack


@dataclass
class AttnWeights:
    """One layer's attention, fp16 row-major as the engine's dense file holds it."""
    input_norm: torch.Tensor | None  # [H]
    q_proj: torch.Tensor             # [heads * dim, H]
    k_proj: torch.Tensor             # [kv_heads * dim, H]
    v_proj: torch.Tensor             # [kv_heads * dim, H]
    o_proj: torch.Tensor             # [H, heads * dim]


def rmsnorm(x: torch.Tensor, w: torch.Tensor | None, eps: float) -> torch.Tensor:
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return y if w is None else y * w.float()


class BatchDecoder:
    #: tokens from which a layer's MoE block takes the tensor-core path
    PREFILL_TOKENS = 96
    #: shared positions from which neighbouring sequences' prefix is read once
    SHARED_POSITIONS = 256

    def __init__(self, stack: MoEStack, layers: list[AttnWeights], embed: torch.Tensor,
                 final_norm: torch.Tensor | None, lm_head: torch.Tensor, n_heads: int,
                 n_kv_heads: int, *, theta: float = 10000.0, scaling: str | None = None,
                 factor: float = 1.0, n_pages: int = 1024, page_size: int = 16, window: int = 0,
                 sinks: int = 0, rows: torch.dtype = torch.float16):
        if len(layers) != stack.L:
            raise ValueError(f"{len(layers)} attention layers for a stack of {stack.L}")
        H = stack.shape.hidden
        if embed.shape[1] != H or H % n_heads or n_heads % n_kv_heads:
            raise ValueError(f"hidden {H}, embedding {list(embed.shape)}, {n_heads} heads, "
                             f"{n_kv_heads} kv heads")
        dim = H // n_heads
        if dim % 16 or dim > 256 or page_size <= 0 or page_size % 8 or window < 0 or sinks < 0:
            raise ValueError(f"heads of {dim} (a multiple of 16 up to 256), page_size {page_size} (of "
                             f"8), window {window}, sinks {sinks} (not negative)")
        if rows not in (torch.float16, torch.float32):
            raise ValueError(f"rows of {rows} (fp16 or fp32)")
        self.rows = rows
        self.stack, self.embed, self.lm_head, self.final_norm = stack, embed, lm_head, final_norm
        self.nh, self.nkv, self.dim = n_heads, n_kv_heads, dim
        self.window, self.sinks, self.eps = window, sinks, stack.shape.rms_eps
        self.device = stack.device
        self.layers = layers
        self._qkv = [torch.cat((w.q_proj, w.k_proj, w.v_proj)) for w in layers]
        self.pool = paged.PagePool(n_pages, page_size)
        shape = (stack.L, n_pages, page_size, n_kv_heads, self.dim)
        self.k = torch.zeros(shape, dtype=torch.float16, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.freq, self.gain = paged.rope_frequencies(self.dim, theta, scaling=scaling,
                                                      factor=factor, device=self.device)

    # ------------------------------------------------------------------ sequences
    def open(self) -> int:
        return self.pool.open()

    def fork(self, seq: int) -> int:
        return self.pool.fork(seq)

    def close(self, seq: int) -> None:
        self.pool.close(seq)

    def truncate(self, seq: int, length: int) -> None:
        """Forget the positions from ``length`` on (rejected drafts, an edited prompt)."""
        self.pool.truncate(seq, length)

    def compact(self) -> int:
        """Move the pages in use to the front of the pools; how many are in use."""
        self.pool.apply(self.k, self.v)  # (what a failed step may have left queued)
        used = self.pool.compact()
        self.pool.apply(self.k, self.v)
        return used

    def _shared(self, seqs: list[int]) -> tuple[list[int], list[int]]:
        """(first sequence of each group and the end, shared positions of each group): runs of
        neighbouring sequences that begin with the same pages."""
        pages = [self.pool.pages(s) for s in seqs]
        page = self.pool.page_size
        starts, lens, i = [0], [], 0
        while i < len(seqs):
            # positions that are in whole pages before every new token: nobody writes them
            common, j = min(len(pages[i]), self.pool.length(seqs[i]) // page), i + 1
            while j < len(seqs):
                n = 0
                while n < min(common, len(pages[j])) and pages[j][n] == pages[i][n]:
                    n += 1
                if n * page < self.SHARED_POSITIONS:
                    break
                common, j = n, j + 1
            starts.append(j)
            lens.append(common * page if j - i > 1 else 0)
            i = j
        return starts, lens

    # ------------------------------------------------------------------ one step
    def step(self, batch: list[tuple[int, list[int]]]) -> torch.Tensor:
        """Append each sequence's tokens; logits fp32 ``[len(batch), vocab]`` of the last ones.

        Waits for the step, and raises where a kernel reported a failure; the sequences are then as
        they were before."""
        if not batch or any(not t for _, t in batch) or len({s for s, _ in batch}) != len(batch):
            raise ValueError("step: each sequence once, with one token or more")
        tokens = [index(t) for _, ts in batch for t in ts]
        for t in tokens:  # (a row that the embedding does not have would fault the GPU)
            if not 0 <= t < self.embed.shape[0]:
                raise ValueError(f"step: token {t} of a vocabulary of {self.embed.shape[0]}")
        before = [(seq, self.pool.length(seq)) for seq, _ in batch]
        try:
            for (seq, n), (_, toks) in zip(before, batch):
                self.pool.extend(seq, n + len(toks))
            self.pool.apply(self.k, self.v)
            return self._run(batch, tokens)
        except BaseException:
            # whatever failed: the lengths must not stand ahead of what has been written
            for seq, n in before:
                self.pool.truncate(seq, n)
            with suppress(Exception):  # pages that got copies keep them
                self.pool.apply(self.k, self.v)
            raise

    def _run(self, batch: list[tuple[int, list[int]]], tokens: list[int]) -> torch.Tensor:
        dev = self.device
        seqs, counts = [s for s, _ in batch], [len(t) for _, t in batch]
        starts = torch.tensor([0] + counts).cumsum(0).to(dev, torch.int32)
        tb = paged.TokenBatch(starts, torch.tensor([self.pool.length(s) for s in seqs],
                                                   dtype=torch.int32, device=dev),
                              self.pool.table(seqs, device=dev), max(counts))
        groups, shared = self._shared(seqs)
        prefix = None
        if any(shared):
            prefix = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (groups, shared)]
        x = self.embed[torch.tensor(tokens, device=dev)].float()
        T, nh, nkv, d = x.shape[0], self.nh, self.nkv, self.dim
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        for l, w in enumerate(self.layers):
            rows = torch.mm(rmsnorm(x, w.input_norm, self.eps).half(), self._qkv[l].T,
                            out_dtype=self.rows)
            q, k, v = (rows[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in
                       ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
            q = paged.rope_append(q, k, v, self.k[l], self.v[l], tb, self.freq, gain=self.gain,
                                  status=status)
            if prefix:
                a = paged.prefix_attention(q, self.k[l], self.v[l], tb, *prefix,
                                           window=self.window, sinks=self.sinks, status=status)
            else:
                a = paged.attention(q, self.k[l], self.v[l], tb, window=self.window,
                                    sinks=self.sinks, status=status)
            x += torch.mm(a.reshape(T, nh * d).half(), w.o_proj.T, out_dtype=torch.float32)
            if T < self.PREFILL_TOKENS:
                self.stack.stack(x, layers=1, layer0=l)
            else:
                x += self.stack.prefill(l, rmsnorm(x, self.stack.layers[l].norm, self.eps))
        last = x[starts[1:].long() - 1]
        logits = torch.mm(rmsnorm(last, self.final_norm, self.eps).half(), self.lm_head.T,
                          out_dtype=torch.float32)
        if bad := status.item():
            raise RuntimeError("step: " + ", ".join(m for b, m in (
                (1, "a page number outside the pool"), (2, "a length beyond the page table"),
                (8, "a wait ran out (paged.wait_limit)")) if bad & b))
        return logits

    def generate(self, seqs: list[int], logits: torch.Tensor, n: int) -> list[list[int]]:
        """``n`` greedy tokens of each sequence, from the logits of its last step on."""
        out: list[list[int]] = [[] for _ in seqs]
        for i in range(n):
            nxt = logits.argmax(-1).tolist()
            for o, t in zip(out, nxt):
                o.append(t)
            if i + 1 < n:
                logits = self.step([(s, [t]) for s, t in zip(seqs, nxt)])
        return out
