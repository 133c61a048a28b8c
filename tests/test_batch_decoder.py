"""BatchDecoder's host side (no GPU): what it refuses, and that a step that fails leaves nothing."""

from types import SimpleNamespace

import pytest
import torch

from wisp_b200 import paged
from wisp_b200.batch_decoder import AttnWeights, BatchDecoder

H, NH, NKV, VOCAB = 128, 2, 1, 50


def decoder(n_heads=NH, n_kv_heads=NKV, **kw):
    """A decoder whose tensors are on the host: a step gets as far as the first operator."""
    d = H // n_heads
    w = AttnWeights(None, torch.zeros(n_heads * d, H).half(), torch.zeros(n_kv_heads * d, H).half(),
                    torch.zeros(n_kv_heads * d, H).half(), torch.zeros(H, n_heads * d).half())
    stack = SimpleNamespace(L=1, shape=SimpleNamespace(hidden=H, rms_eps=1e-6),
                            device=torch.device("cpu"), layers=[None])
    return BatchDecoder(stack, [w], torch.zeros(VOCAB, H).half(), None,
                        torch.zeros(VOCAB, H).half(), n_heads, n_kv_heads, n_pages=16, **kw)


@pytest.mark.parametrize("tokens", [[VOCAB], [3, -1], [1 << 40]])
def test_tokens_outside_the_vocabulary_are_refused(built_lib, tokens):
    dec = decoder()
    s = dec.open()
    with pytest.raises(ValueError, match="of a vocabulary of 50"):
        dec.step([(s, tokens)])
    assert dec.pool.length(s) == 0 and dec.pool.free_pages == 16


def test_a_step_that_fails_leaves_the_lengths(built_lib):
    """Here the first operator refuses host tensors; before it and behind it anything may fail."""
    dec = decoder()
    a, b = dec.open(), dec.open()
    with pytest.raises(ValueError, match="CUDA tensor"):
        dec.step([(a, [1, 2, 3]), (b, [4] * 40)])
    assert dec.pool.length(a) == dec.pool.length(b) == 0 and dec.pool.free_pages == 16
    for bad in ([1.5], ["x"], [None]):
        with pytest.raises(TypeError):
            dec.step([(a, [1]), (b, bad)])
    assert dec.pool.length(a) == dec.pool.length(b) == 0 and dec.pool.free_pages == 16


def test_an_interrupted_step_keeps_a_fork_apart(built_lib, monkeypatch):
    """The page that a fork was about to write stays its own, and its copy is made."""
    dec = decoder()
    a = dec.open()
    dec.pool.extend(a, 20)
    b = dec.fork(a)
    made = []
    monkeypatch.setattr(paged, "copy_pages", lambda k, v, s, d: made.append((list(s), list(d))))

    def stop(*_):
        raise KeyboardInterrupt

    monkeypatch.setattr(paged, "TokenBatch", stop)
    with pytest.raises(KeyboardInterrupt):
        dec.step([(b, [1, 2])])
    assert dec.pool.length(a) == dec.pool.length(b) == 20
    assert dec.pool.pages(a) == [0, 1] and dec.pool.pages(b) == [0, 2]
    assert made == [([1], [2])] and dec.pool.moves() == ([], [])


@pytest.mark.parametrize("kw,msg", [(dict(page_size=12), "page_size 12"), (dict(page_size=0), "page_size"),
                                    (dict(n_heads=16, n_kv_heads=2), "heads of 8"),
                                    (dict(window=-1), "window -1"), (dict(sinks=-3), "sinks -3")])
def test_shapes_that_the_operators_refuse_are_refused_at_once(built_lib, kw, msg):
    with pytest.raises(ValueError, match=msg):
        decoder(**kw)


def test_rows_of_other_types_are_refused(built_lib):
    with pytest.raises(ValueError, match="rows of torch.bfloat16"):
        decoder(rows=torch.bfloat16)
