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
