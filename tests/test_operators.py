"""The operators that make the gradient, without a GPU: what they refuse (before anything is launched), and the sizes of
their workspaces."""
import os
import subprocess

import pytest
import torch

from omr import _lib, ops

EINVAL = _lib.OMR_EINVAL
A = 1 << 12  # an address that is only checked


def refused(rc, text):
    assert rc == EINVAL
    assert text in _lib.load().omr_last_error().decode(), _lib.load().omr_last_error()


def embed(**k):
    a = dict(table=A, td=1, rows=10, dim=8, stride=8, ids=A, ids64=1, n=4, scale=1.0, out=A, od=1, ostride=8)
    a.update(k)
    return _lib.load().omr_embed(*a.values(), None)


def embed_grad(**k):
    a = dict(grad=A, gd=1, gstride=8, ids=A, ids64=1, n=4, rows=10, dim=8, scale=1.0, out=A, ostride=8, acc=0, ws=A,
             bytes=1 << 30)
    a.update(k)
    return _lib.load().omr_embed_grad_f32(*a.values(), None)


def norm(**k):
    a = dict(x=A, dt=1, rows=4, dim=8, stride=8, w=A, b=A, pdt=0, eps=1e-5, out=A, ostride=8, mean=A, rstd=A)
    a.update(k)
    return _lib.load().omr_layer_norm(*a.values(), None)


def norm_grad(**k):
    a = dict(dy=A, dystride=8, x=A, dt=1, rows=4, dim=8, stride=8, mean=A, rstd=A, w=A, pdt=0, dx=A, dxstride=8, dw=A, db=A,
             acc=0, ws=A, bytes=1 << 30)
    a.update(k)
    return _lib.load().omr_layer_norm_grad(*a.values(), None)


def loss(**k):
    a = dict(h=A, hs=8, w=A, wstride=8, dt=1, n=4, vocab=10, dim=8, t=A, t64=1, loss=A, lse=A, ws=A, bytes=1 << 40)
    a.update(k)
    return _lib.load().omr_vocab_loss(*a.values(), None)


def loss_grad(**k):
    a = dict(h=A, hs=8, w=A, wstride=8, dt=1, n=4, vocab=10, dim=8, t=A, t64=1, lse=A, g=A, gs=1, gh=A, ghs=8, gw=A, gwd=0,
             gws=8, acc=0, ws=A, bytes=1 << 40)
    a.update(k)
    return _lib.load().omr_vocab_loss_grad(*a.values(), None)


@pytest.mark.parametrize("call,arg,text", [
    (embed, dict(td=3), "element type"), (embed, dict(od=-1), "element type"), (embed, dict(dim=0), "dim"),
    (embed, dict(dim=(1 << 24) + 1, ostride=1 << 25), "dim"), (embed, dict(rows=1 << 31), "2^31"),
    (embed, dict(n=1 << 31), "2^31"), (embed, dict(ostride=7), "stride"), (embed, dict(out=None), "NULL"),
    (embed, dict(ids=None), "NULL"), (embed, dict(table=None), "NULL"),
    (embed, dict(n=(1 << 31) - 1, dim=1 << 16, ostride=1 << 16), "too many"),
    (embed_grad, dict(gd=5), "element type"), (embed_grad, dict(dim=0), "dim"), (embed_grad, dict(rows=1 << 31), "2^31"),
    (embed_grad, dict(n=1 << 31), "2^31"), (embed_grad, dict(ostride=4), "stride"), (embed_grad, dict(out=None), "NULL"),
    (embed_grad, dict(ws=None), "NULL"), (embed_grad, dict(ids=None), "NULL"), (embed_grad, dict(ws=A + 8), "aligned"),
    (embed_grad, dict(bytes=16), "workspace of 16 bytes"),
    (norm, dict(dt=4), "elements"), (norm, dict(pdt=2), "parameters"), (norm, dict(dim=0), "dim"),
    (norm, dict(ostride=7), "stride"), (norm, dict(eps=-1.0), "eps"), (norm, dict(eps=float("nan")), "eps"),
    (norm, dict(mean=None), "NULL"), (norm, dict(x=None), "NULL"),
    (norm_grad, dict(dt=7), "elements"), (norm_grad, dict(pdt=2), "parameters"), (norm_grad, dict(dxstride=1), "stride"),
    (norm_grad, dict(dx=None), "NULL"), (norm_grad, dict(rstd=None), "NULL"), (norm_grad, dict(ws=None), "workspace"),
    (norm_grad, dict(ws=A + 4), "aligned"), (norm_grad, dict(bytes=0), "workspace of 0 bytes"),
    (loss, dict(dt=0), "bf16 or fp16"), (loss, dict(dim=0), "dim"), (loss, dict(dim=(1 << 20) + 1), "dim"),
    (loss, dict(vocab=0), "vocab"), (loss, dict(vocab=1 << 31), "vocab"), (loss, dict(n=1 << 31), "tokens"),
    (loss, dict(n=1 << 26), "2^26"), (loss_grad, dict(n=1 << 26), "2^26"),
    (embed_grad, dict(n=(1 << 31) - 1, bytes=1 << 50), "too many"),
    (loss, dict(t=None), "NULL"), (loss, dict(lse=None), "NULL"), (loss, dict(ws=None), "workspace"),
    (loss, dict(bytes=100), "workspace of 100 bytes"), (loss, dict(wstride=9, bytes=(4 << 20) + 1100), "pack"),
    (loss, dict(w=A + 2, bytes=(4 << 20) + 1100), "pack"),
    (loss_grad, dict(dt=0), "bf16 or fp16"), (loss_grad, dict(gwd=2), "grad_weight"), (loss_grad, dict(ghs=7), "stride"),
    (loss_grad, dict(gws=7), "stride"), (loss_grad, dict(g=None), "NULL"), (loss_grad, dict(lse=None), "NULL"),
    (loss_grad, dict(bytes=1000), "workspace of 1000 bytes"),
])
def test_refusals(call, arg, text):
    refused(call(**arg), text)


def test_empty_calls_launch_nothing():
    assert embed(n=0, ids=None, out=None) == 0
    assert embed_grad(rows=0, out=None, ws=None) == 0
    assert norm(rows=0, x=None, out=None) == 0
    assert loss(n=0, h=None, ws=None) == 0
    assert loss_grad(n=0, gw=None) == 0
    assert loss_grad(n=0, acc=1) == 0


def test_workspaces_grow_with_the_call():
    """A plan for so many tokens holds any smaller call."""
    lib = _lib.load()
    for size in (lambda n: lib.omr_embed_grad_workspace_bytes(n, 5000, 300),
                 lambda n: lib.omr_layer_norm_grad_workspace_bytes(n, 300),
                 lambda n: lib.omr_vocab_loss_workspace_bytes(n, 50001, 300, 1, 1),
                 lambda n: lib.omr_vocab_loss_workspace_bytes(n, 50001, 300, 0, 0),
                 lambda n: lib.omr_vocab_loss_workspace_bytes(n, 1 << 30, 64, 0, 1)):
        at = [size(n) for n in (0, 1, 2, 15, 16, 17, 31, 33, 100, 257, 1000, 2048, 4095, 5000, 20000, 100000)]
        assert at == sorted(at) and at[-1] < 1 << 50


def test_the_front_end_refuses():
    t = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="device"):
        ops.embed(t, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="device"):
        ops.layer_norm(t)
    with pytest.raises(ValueError, match="dtype"):
        ops.VocabLossPlan(4, 10, 8, dtype=torch.float32)
    with pytest.raises(ValueError, match="sizes"):
        ops.VocabLossPlan(4, 0, 8)
    for make in (lambda: ops.EmbedGradPlan(-1, 10, 8), lambda: ops.EmbedGradPlan(4, 1 << 31, 8),
                 lambda: ops.EmbedGradPlan(4, 10, (1 << 32) + 8), lambda: ops.LayerNormGradPlan(-2, 8),
                 lambda: ops.LayerNormGradPlan(4, 0), lambda: ops.VocabLossPlan(4, -1, 8),
                 lambda: ops.VocabLossPlan(4, 10, 1 << 40)):
        with pytest.raises(ValueError, match="sizes"):
            make()


@pytest.mark.parametrize("call,arg", [
    (loss, dict(n=1 << 25, vocab=1 << 20)),                      # 2^17 x 2^12 tiles
    (loss, dict(n=1 << 25, vocab=1 << 20, wstride=9)),           # and rows to be laid out first
    (loss, dict(vocab=(1 << 31) - 300)),                         # a few tokens, 2^25 workgroups
    (loss, dict(n=4, vocab=(1 << 31) - 300, wstride=9)),
    (loss, dict(n=(1 << 26) - 2, vocab=10)),                     # 2^24 workgroups that join
    (loss_grad, dict(n=1 << 25, dim=1 << 20, hs=1 << 20, wstride=1 << 20, ghs=1 << 20, gws=1 << 20)),  # grad_hidden's tiles
    (loss_grad, dict(n=1 << 25, dim=1 << 20, hs=1 << 20, wstride=1 << 20, ghs=1 << 20, gw=None)),
    (loss_grad, dict(vocab=(1 << 31) - 300, dim=1001, hs=1001, wstride=1001, ghs=1001, gws=1001)),  # 2^29 that lay out rows
    (loss_grad, dict(n=(1 << 26) - 1, vocab=1 << 29, dim=1 << 10, hs=1 << 10, wstride=1 << 10, ghs=1 << 10, gws=1 << 10)),
])
def test_sizes_no_launch_takes_are_refused_first(call, arg):
    """Before anything is launched, the laying out of rows and the sort among it: without a GPU a launch would say that there
    is none."""
    refused(call(**{"bytes": 1 << 62, **arg}), "too many")


def test_workspaces_of_sizes_no_call_takes():
    """Are 0 bytes, and no plan is made for them: their products would pass 64 bits (2^40 tokens of 2^24), and a plan's first
    call would be refused."""
    lib = _lib.load()
    for size in (lib.omr_vocab_loss_workspace_bytes(1 << 26, 100, 64, 0, 1),
                 lib.omr_vocab_loss_workspace_bytes(1 << 39, 100, 1 << 24, 0, 1),
                 lib.omr_vocab_loss_workspace_bytes(10, 100, (1 << 20) + 1, 0, 1),
                 lib.omr_vocab_loss_workspace_bytes(10, (1 << 31) - 256, 64, 0, 1),
                 lib.omr_vocab_loss_workspace_bytes(10, 0, 64, 0, 1), lib.omr_vocab_loss_workspace_bytes(10, 9, 0, 0, 1),
                 lib.omr_embed_grad_workspace_bytes(1 << 31, 10, 8), lib.omr_embed_grad_workspace_bytes(10, 1 << 31, 8),
                 lib.omr_embed_grad_workspace_bytes(10, 10, (1 << 24) + 1), lib.omr_embed_grad_workspace_bytes(10, 10, 0),
                 lib.omr_layer_norm_grad_workspace_bytes(1 << 40, 8), lib.omr_layer_norm_grad_workspace_bytes(8, 0),
                 lib.omr_layer_norm_grad_workspace_bytes(8, (1 << 24) + 1)):
        assert size == 0
    for least in (lib.omr_vocab_loss_workspace_bytes(0, 1, 1, 0, 0), lib.omr_embed_grad_workspace_bytes(0, 0, 1),
                  lib.omr_layer_norm_grad_workspace_bytes(0, 1)):
        assert least >= 16
    for make in (lambda: ops.VocabLossPlan(1 << 26, 100, 64, device="cpu"),
                 lambda: ops.VocabLossPlan(1 << 39, 100, 1 << 24, device="cpu"),
                 lambda: ops.VocabLossPlan(4, 10, (1 << 20) + 8, device="cpu"),
                 lambda: ops.EmbedGradPlan(1 << 31, 10, 8, device="cpu")):
        with pytest.raises(ValueError, match="sizes"):
            make()


@pytest.mark.parametrize("value", ["4294967304:5", "8:5x", "8x:5", "-8:5", "8:-5", "8:", ":5", "8", "", "0:5", "8:0",
                                   "8:18446744073709551617", "12:5", "56:5", "8:1073741824", "1048584:5"])
def test_the_client_refuses_sizes(value):
    """./omr_client -E <dim>:<tokens>, before it looks for a device: numbers that are not two of their range, or no
    multiple of 8 that divides the tensor."""
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omnireduce-rdma-demo_amd", "bin",
                       "omr_client")
    p = subprocess.run([exe, "-L", "1", "-n", str(1048584 << 4), "-E", value], capture_output=True, text=True, timeout=60)
    assert p.returncode == 1 and "-E" in p.stderr and "device" not in p.stderr, p.stderr
