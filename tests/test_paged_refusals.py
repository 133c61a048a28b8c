"""Arguments of the paged cache's calls that are refused before any GPU work (no GPU)."""

import ctypes as C

import pytest
import torch

from wisp_b200 import paged
from wisp_b200.lib import WispErrCtx, WispKvPages, WispRows, WispTokenBatch, lib


def attention(q, out, tokens=7, **batch):
    """The refusal of a call without a workspace, which is looked at last."""
    P = WispKvPages(1024, 2048, 16 * 2 * 64, 4, 16, 2, 64, 1)
    B = WispTokenBatch(**dict(dict(q_start=64, kv_len=64, table=64, n_seq=2, n_tokens=tokens, max_q=7,
                                   table_stride=4), **batch))
    err = WispErrCtx()
    rc = lib().wisp_paged_attention(C.byref(q), C.byref(out), None, C.byref(P), C.byref(B),
                                    C.c_float(0.1), 0, 0, None, 0, None, C.byref(err))
    assert rc == 4
    return err.message.decode()


ROW = 8 * 64  # elements of a row of 8 heads


@pytest.mark.parametrize("at,stride,tokens,over", [
    (0, ROW, 7, True), (ROW, ROW, 7, True), (6 * ROW, ROW, 7, True), (7 * ROW, ROW, 7, False),
    (-7 * ROW, ROW, 7, False), (-7 * ROW + 8, ROW, 7, True), (0, ROW, 1, True), (ROW, ROW, 1, False),
    (ROW, 2 * ROW, 7, True)])
def test_out_must_not_overlap_q(built_lib, at, stride, tokens, over):
    base = 1 << 20
    msg = attention(WispRows(base, ROW, 8, 1), WispRows(base + 2 * at, stride, 8, 1), tokens)
    assert ("overlap" if over else "workspace") in msg, msg


@pytest.mark.parametrize("at,width,out_stride,over", [
    (ROW, 3 * ROW, 3 * ROW, False), (2 * ROW, 3 * ROW, 3 * ROW, False), (ROW - 8, 3 * ROW, 3 * ROW, True),
    (2 * ROW + 8, 3 * ROW, 3 * ROW, True), (ROW, 2 * ROW, 4 * ROW, False), (ROW, 4 * ROW, 2 * ROW, False),
    (ROW, 2 * ROW, 3 * ROW, True)])
def test_out_and_q_may_lie_beside_each_other(built_lib, at, width, out_stride, over):
    """Columns of one buffer of rows (a fused projection), and rows between rows."""
    base = 1 << 20
    msg = attention(WispRows(base, width, 8, 1), WispRows(base + 2 * at, out_stride, 8, 1))
    assert ("overlap" if over else "workspace") in msg, msg


# ------------------------------------------------------------------------ gradients
def test_pages_that_ask_for_a_gradient_are_refused():
    plain = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    asks = plain.clone().requires_grad_()
    q = torch.zeros(2, 8, 64, dtype=torch.float16)
    for k, v, name in ((asks, plain, "k_pages"), (plain, asks, "v_pages")):
        for call in (lambda: paged.attention(q, k, v, None), lambda: paged.copy_pages(k, v, [0], [1])):
            with pytest.raises(ValueError, match=name + " asks for a gradient"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
                call()


def test_forward_mode_tangents_are_refused():
    plain = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    q = torch.zeros(2, 8, 64, dtype=torch.float16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(plain, torch.ones_like(plain))
        for k, v, name in ((dual, plain, "k_pages"), (plain, dual, "v_pages")):
            with torch.no_grad(), pytest.raises(ValueError, match=name + " has a forward-mode tangent"):
                paged.attention(q, k, v, None)
    with pytest.raises(ValueError, match="CUDA device"):
        paged.attention(q, plain, plain, None)


# ------------------------------------------------------------------------ calls too long for 32 bits
@pytest.mark.parametrize("tokens,heads,window,long", [
    (1 << 20, 64, 0, True), (1 << 20, 64, 4096, False), (1 << 20, 8, 0, False), (8192, 64, 0, False),
    (1 << 22, 64, 1 << 20, True)])
def test_a_prompt_whose_work_passes_31_bits_is_refused(built_lib, tokens, heads, window, long):
    """One kv head, a table of 2^20 positions: the row tiles' KV tiles are counted in 32 bits."""
    P = WispKvPages(1024, 2048, 16 * 64, 1 << 20, 16, 1, 64, 1)
    B = WispTokenBatch(64, 64, 64, 1, tokens, tokens, 1 << 16, 0)
    q, out = WispRows(1 << 20, heads * 64, heads, 1), WispRows(1 << 40, heads * 64, heads, 1)
    err = WispErrCtx()
    rc = lib().wisp_paged_attention(C.byref(q), C.byref(out), None, C.byref(P), C.byref(B),
                                    C.c_float(0.1), window, 0, None, 0, None, C.byref(err))
    assert rc == 4 and ("in one call" if long else "workspace") in err.message.decode(), err.message
