"""The batched decoder (paged cache, rotary append, attention, MoE) against the one-sequence
decoder step (wisp_attn_decode on a contiguous cache, token by token) on the same weights.

Tolerance: the batched form rounds the projections' inputs and outputs and the attention rows to
fp16 where the one-sequence step keeps fp32: a few 2^-11 per layer, so logits within rel-L2 1e-2
(the output bound of the other decoder tests).  Every token's experts are all of the layer's, so
that no near-tie of the router changes the comparison.
"""

import ctypes as C

import numpy as np
import pytest
import torch

from wisp_b200 import converter as cv
from wisp_b200.batch_decoder import AttnWeights, BatchDecoder
from wisp_b200.lib import WispAttnLayer, WispErrCtx, check, lib
from wisp_b200.moe import MoEStack

pytestmark = pytest.mark.gpu

H, NH, NKV, L, VOCAB = 512, 8, 2, 2, 300


@pytest.fixture(scope="module")
def model(cuda):
    stack = MoEStack(cv.MoEShape(hidden=H, inter=512, n_experts=2, top_k=2, n_layers=L), seed=3,
                     device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)

    def w(*shape, s=1.0):
        return (torch.randn(*shape, generator=g, device=cuda) * s).half()

    d = H // NH
    layers = [AttnWeights((1 + 0.1 * w(H).float()).half(), w(NH * d, H, s=H ** -0.5),
                          w(NKV * d, H, s=H ** -0.5), w(NKV * d, H, s=H ** -0.5),
                          w(H, NH * d, s=(NH * d) ** -0.5)) for _ in range(L)]
    return stack, layers, w(VOCAB, H), (1 + 0.1 * w(H).float()).half(), w(VOCAB, H, s=H ** -0.5)


def decoder(model, **kw):
    stack, layers, embed, norm, head = model
    return BatchDecoder(stack, layers, embed, norm, head, NH, NKV, n_pages=128, **kw)


def one_by_one(model, tokens):
    """Logits after each token from the fused one-token layers."""
    stack, layers, embed, norm, head = model
    dev, d, seq = stack.device, H // NH, 1024
    s = torch.cuda.current_stream().cuda_stream
    kv = [[torch.zeros(seq, NKV, d, dtype=torch.float16, device=dev) for _ in range(2)]
          for _ in range(L)]
    A = [WispAttnLayer(w.input_norm.data_ptr(), w.q_proj.data_ptr(), w.k_proj.data_ptr(),
                       w.v_proj.data_ptr(), w.o_proj.data_ptr(), H, NH, NKV, d, 10000.0,
                       stack.shape.rms_eps) for w in layers]
    n = int(lib().wisp_attn_workspace_bytes(C.byref(A[0]), seq))
    ws = torch.zeros(n, dtype=torch.uint8, device=dev)
    out, err = [], WispErrCtx()
    tmp = torch.empty(H, device=dev)
    for pos, t in enumerate(tokens):
        x = embed[t].float()[None].contiguous()
        for l in range(L):
            check(lib().wisp_attn_decode(C.byref(A[l]), x.data_ptr(), kv[l][0].data_ptr(),
                                         kv[l][1].data_ptr(), pos, seq, ws.data_ptr(), n, s,
                                         C.byref(err)), err)
            stack.stack(x, layers=1, layer0=l)
        y = torch.empty(VOCAB, device=dev)
        check(lib().wisp_lm_head_forward(norm.data_ptr(), head.data_ptr(), x.data_ptr(),
                                         y.data_ptr(), VOCAB, H, stack.shape.rms_eps,
                                         tmp.data_ptr(), tmp.numel() * 4, s, C.byref(err)), err)
        out.append(y)
    return torch.stack(out)


def close(got, want):
    rel = (got - want).norm() / want.norm()
    assert rel <= 1e-2, rel.item()


def prompt(n, seed):
    return np.random.default_rng(seed).integers(0, VOCAB, n).tolist()


def test_prompts_chunks_and_single_tokens_in_one_batch(model):
    a, b, c = prompt(150, 1), prompt(23, 2), prompt(41, 3)
    want = {k: one_by_one(model, v) for k, v in (("a", a), ("b", b), ("c", c))}
    dec = decoder(model)
    sa, sb, sc = dec.open(), dec.open(), dec.open()
    close(dec.step([(sa, a[:1])]), want["a"][:1])
    close(dec.step([(sb, b[:7]), (sa, a[1:100])]),           # a prompt behind a chunk
          torch.stack((want["b"][6], want["a"][99])))
    got = dec.step([(sa, a[100:149]), (sc, c[:40]), (sb, b[7:8])])
    close(got, torch.stack((want["a"][148], want["c"][39], want["b"][7])))
    got = dec.step([(sb, b[8:22]), (sc, c[40:])])
    close(got, torch.stack((want["b"][21], want["c"][40])))
    got = dec.step([(sa, a[149:]), (sb, b[22:])])
    close(got, torch.stack((want["a"][149], want["b"][22])))


def test_truncated_and_compacted_sequences_go_on(model):
    a, b = prompt(60, 4), prompt(30, 5)
    want = one_by_one(model, a)
    dec = decoder(model)
    sb, sa = dec.open(), dec.open()
    dec.step([(sb, b), (sa, a[:40] + prompt(9, 6))])   # nine tokens that are rejected
    dec.truncate(sa, 40)
    dec.close(sb)
    assert dec.compact() == 3
    close(dec.step([(sa, a[40:])]), want[59:60])


def test_answers_behind_a_shared_prefix(model):
    """Four answers to one prompt: the shared pages are read once, and each answer is what its
    tokens alone give."""
    p = prompt(400, 7)
    dec = decoder(model)
    first = dec.open()
    logits = dec.step([(first, p)])
    seqs = [first] + [dec.fork(first) for _ in range(3)]
    tails = [prompt(3, 10 + i) for i in range(4)]
    assert dec._shared(seqs)[0] == [0, 4]
    for i in range(3):
        got = dec.step([(s, [t[i]]) for s, t in zip(seqs, tails)])
        assert dec._shared(seqs) == ([0, 4], [400])
    want = torch.stack([one_by_one(model, p + t)[-1] for t in tails])
    close(got, want)
    alone = decoder(model)
    alone.SHARED_POSITIONS = 1 << 30
    s0 = alone.open()
    close(alone.step([(s0, p)]), logits)
    others = [s0] + [alone.fork(s0) for _ in range(3)]
    for i in range(3):
        plain = alone.step([(s, [t[i]]) for s, t in zip(others, tails)])
    close(plain, got)


def test_window_and_sinks_forget_the_middle(model):
    """With a window, tokens that no layer's window reaches change nothing; the sinks do."""
    p = prompt(300, 8)
    dec = decoder(model, window=32, sinks=2)
    other = list(p)
    other[100:140] = prompt(40, 9)
    start = list(p)
    start[0] = (p[0] + 1) % VOCAB
    seqs = [dec.open() for _ in range(3)]
    got = dec.step([(s, t) for s, t in zip(seqs, (p, other, start))])
    assert torch.equal(got[0], got[1]) or (got[0] - got[1]).norm() <= 1e-3 * got[0].norm()
    assert (got[0] - got[2]).norm() > 1e-2 * got[0].norm()


def test_generate_and_refusals(model):
    dec = decoder(model)
    s = dec.open()
    logits = dec.step([(s, prompt(5, 11))])
    out = dec.generate([s], logits, 4)
    assert len(out) == 1 and len(out[0]) == 4 and dec.pool.length(s) == 8
    with pytest.raises(ValueError, match="each sequence once"):
        dec.step([(s, [1]), (s, [2])])
    with pytest.raises(ValueError, match="one token or more"):
        dec.step([(s, [])])
    other, free = dec.open(), dec.pool.free_pages
    with pytest.raises(RuntimeError, match="pages needed"):
        dec.step([(other, [1]), (s, prompt(16 * 128, 1))])
    assert dec.pool.length(s) == 8 and dec.pool.length(other) == 0
    assert dec.pool.free_pages == free
