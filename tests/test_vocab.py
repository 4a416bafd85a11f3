"""The vocabulary operators without a GPU: refusals of the Python calls and of the C entries, workspace queries."""
import ctypes as C

import pytest
import torch

from gossipnet_amd import _lib, vocab

F32, BF16 = 0, 1


def xent_args(M=4, V=10, D=8, dtype=torch.float32):
    return torch.zeros(M, D, dtype=dtype), torch.zeros(V, D, dtype=dtype), torch.zeros(M, dtype=torch.int64)


def test_cpu_tensors_are_refused():
    x, w, y = xent_args()
    one = torch.zeros(4)
    for call in (lambda: vocab.xent_forward(x, w, y), lambda: vocab.xent_backward(x, w, y, one, one, one),
                 lambda: vocab.distill_forward(x, w, y[:, None], one[:, None]), lambda: vocab.embed_forward(y, w),
                 lambda: vocab.distill_backward(x, w, y[:, None], one[:, None], one, one[:, None], one), lambda: vocab.embed_backward(y, x, w)):
        with pytest.raises(_lib.GnetError, match="device kernels"):
            call()


@pytest.mark.parametrize("change, match", [
    (dict(x=torch.zeros(4, 9)), "columns"), (dict(x=torch.zeros(4, 8, dtype=torch.float16)), "float16"),
    (dict(x=torch.zeros(4, 8, dtype=torch.float64)), "float32, bfloat16 or float16"), (dict(x=torch.tensor(1.)), "at least one dimension"),
    (dict(w=torch.zeros(8)), "V >= 1"), (dict(w=torch.zeros(0, 8)), "V >= 1"), (dict(w=torch.zeros(10, 0), x=torch.zeros(4, 0)), "no elements"),
    (dict(labels=torch.zeros(5, dtype=torch.int64)), "shape"), (dict(labels=torch.zeros(4)), "int32 or int64"),
    (dict(labels=torch.zeros(4, 1, dtype=torch.int64)), "shape")])
def test_xent_refusals(change, match):
    x, w, y = xent_args()
    a = dict(x=x, w=w, labels=y)
    a.update(change)
    with pytest.raises(_lib.InvalidArgumentError, match=match):
        vocab.xent_forward(**a)
    one = torch.zeros(4)
    with pytest.raises(_lib.InvalidArgumentError, match=match):
        vocab.xent_backward(a["x"], a["w"], a["labels"], one, one, one)


def test_backward_refuses_statistics_of_other_shapes():
    x, w, y = xent_args()
    one, bad = torch.zeros(4), torch.zeros(3)
    for lse, hit, g in ((bad, one, one), (one, bad, one), (one, one, bad), (one, one, torch.zeros(1))):
        with pytest.raises(_lib.InvalidArgumentError, match="shape"):
            vocab.xent_backward(x, w, y, lse, hit, g)
    ids, t = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    with pytest.raises(_lib.InvalidArgumentError, match="hit has shape"):
        vocab.distill_backward(x, w, ids, t, one, one, one)


@pytest.mark.parametrize("ids, logits, temperature, match", [
    (torch.zeros(4, 0, dtype=torch.int32), torch.zeros(4, 0), 1.0, "K >= 1"), (torch.zeros(4, dtype=torch.int32), torch.zeros(4), 1.0, "K >= 1"),
    (torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2), 1.0, "tokens"), (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 3), 1.0, "shape"),
    (torch.zeros(4, 2, dtype=torch.int16), torch.zeros(4, 2), 1.0, "int32 or int64"), (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), 0.0, "temperature"),
    (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), -1.0, "temperature"),
    (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), float("nan"), "temperature"),
    (torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), float("inf"), "temperature")])
def test_distill_refusals(ids, logits, temperature, match):
    x, w, _ = xent_args()
    with pytest.raises(_lib.InvalidArgumentError, match=match):
        vocab.distill_forward(x, w, ids, logits, temperature)


def test_embed_refusals():
    t, ids, dy = torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8)
    bad = [lambda: vocab.embed_forward(ids, torch.zeros(8)), lambda: vocab.embed_forward(ids, torch.zeros(0, 8)),
           lambda: vocab.embed_forward(ids.float(), t), lambda: vocab.embed_forward(ids, t.double()),
           lambda: vocab.embed_forward(ids, t, 1.0, torch.zeros(5)), lambda: vocab.embed_backward(ids, dy[:3], t),
           lambda: vocab.embed_backward(ids, dy.half(), t), lambda: vocab.embed_backward(ids, dy, t, out=torch.zeros(10, 7)),
           lambda: vocab.embed_backward(ids, dy, t, out=torch.zeros(10, 8, dtype=torch.float16)),
           lambda: vocab.embed_backward(ids, dy, t, out=torch.zeros(8, 10).t())]
    for call in bad:
        with pytest.raises(_lib.InvalidArgumentError):
            call()


def test_c_entries_refuse_before_they_launch():
    """Bad sizes, types, pointers and workspaces come back as a status; nothing is launched (the pointers are never followed)."""
    lib = _lib.load()
    p, odd = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 8)

    def xent(x=p, ldx=8, w=p, ldw=8, y=p, M=4, V=10, D=8, dtype=F32, loss=p, ws=p, n=1 << 40):
        return lib.gnet_xent_forward(x, ldx, w, ldw, y, 1, M, V, D, dtype, loss, p, p, ws, n, None)

    def xent_back(lse=p, g=p, M=4, n=1 << 40):
        return lib.gnet_xent_backward(p, 8, p, 8, p, 1, lse, p, g, M, 10, 8, F32, p, p, p, n, None)
    for a in (dict(M=-1), dict(V=0), dict(D=0), dict(ldx=7), dict(ldw=7), dict(dtype=3), dict(x=None), dict(w=None), dict(y=None), dict(loss=None)):
        assert xent(**a) == _lib.ERR_INVALID, a
    for a in (dict(M=(1 << 24) + 1), dict(V=(1 << 30) + 1), dict(D=(1 << 16) + 1, ldx=1 << 17, ldw=1 << 17), dict(M=1 << 24, V=1 << 21)):
        assert xent(**a) == _lib.ERR_UNSUPPORTED, a
    assert lib.gnet_vocab_workspace_bytes(p, 8, 4, 10, 8, 0, F32, 0) == 0           # (a small vocabulary's forward pass keeps nothing)
    for M, V in ((4, 3000), (100, 3000), (9000, 10)):
        need = lib.gnet_vocab_workspace_bytes(p, 8, M, V, 8, 0, F32, 0)
        assert need > 0
        for a in (dict(ws=None), dict(n=need - 1), dict(ws=odd)):
            assert xent(M=M, V=V, **a) == _lib.ERR_WORKSPACE, a
    assert xent_back(lse=None) == xent_back(g=None) == _lib.ERR_INVALID
    assert xent_back(n=16) == _lib.ERR_WORKSPACE
    assert xent(M=0, x=None, y=None, loss=None, ws=None, n=0) == _lib.OK

    def distill(K=2, temperature=1.0, logits=p):
        return lib.gnet_distill_forward(p, 8, p, 8, p, 0, logits, temperature, 4, 10, 8, K, F32, p, p, p, p, 1 << 40, None)
    for a in (dict(K=0), dict(temperature=0.0), dict(temperature=-2.0), dict(temperature=float("nan")), dict(logits=None)):
        assert distill(**a) == _lib.ERR_INVALID, a
    assert distill(K=1025) == _lib.ERR_UNSUPPORTED

    def embed(ids=p, ld=8, M=4, V=10, D=8, dtype=BF16, out=p, table=p, ld_table=8, dscale=p, ws=p, n=1 << 30):
        return lib.gnet_embed_backward(ids, 0, p, ld, 1.0, None, M, V, D, dtype, out, 0, table, ld_table, dscale, ws, n, None)
    for a in (dict(M=-1), dict(V=0), dict(D=0), dict(ld=7), dict(dtype=-1), dict(ids=None), dict(out=None), dict(table=None), dict(ld_table=7)):
        assert embed(**a) == _lib.ERR_INVALID, a
    assert lib.gnet_embed_workspace_bytes(64, 8) == 0 < lib.gnet_embed_workspace_bytes(65, 8)
    for a in (dict(ws=None), dict(n=8), dict(ws=odd)):
        assert embed(M=65, V=3000, **a) == _lib.ERR_WORKSPACE and embed(M=65, **a) == _lib.ERR_WORKSPACE, a
    assert lib.gnet_embed_forward(p, 0, p, 7, 1.0, None, 4, 10, 8, BF16, p, None) == _lib.ERR_INVALID
    assert lib.gnet_embed_forward(None, 0, p, 8, 1.0, None, 4, 10, 8, BF16, p, None) == _lib.ERR_INVALID
    assert lib.gnet_embed_forward(None, 0, None, 8, 1.0, None, 0, 10, 8, BF16, None, None) == _lib.OK


def test_workspaces_do_not_grow_with_the_logits():
    """The backward pass keeps one piece of the vocabulary: its scratch stays far below the M x V logits."""
    lib = _lib.load()
    p = C.c_void_p(1 << 20)
    M, V, D = 4096, 131072, 4096
    assert lib.gnet_vocab_workspace_bytes(p, D, M, V, D, 0, BF16, 1) < M * V
    assert lib.gnet_vocab_workspace_bytes(p, D, M, V, D, 0, BF16, 0) < M * V // 4
    assert lib.gnet_vocab_workspace_bytes(p, D, 0, V, D, 0, BF16, 0) == 0
    # a weight matrix that cannot be read where it lies is packed: only then is there room for it
    assert lib.gnet_vocab_workspace_bytes(C.c_void_p((1 << 20) + 2), D, 64, V, D, 0, BF16, 0) > lib.gnet_vocab_workspace_bytes(p, D, 64, V, D, 0, BF16, 0)


def test_few_tokens_lay_no_weights_out():
    """fp32 weights and odd widths are copied for many tokens only; both workspaces are checked."""
    lib = _lib.load()
    p = C.c_void_p(1 << 20)
    V, D = 100000, 2047
    for dtype, size in ((F32, 4), (BF16, 2)):
        for backward in (0, 1):
            few, many = (lib.gnet_vocab_workspace_bytes(p, D, M, V, D, 0, dtype, backward) for M in (32, 33))
            assert 0 < few < V * D * size // 4 and few < many, (dtype, backward)
        for M in (32, 33):
            need = lib.gnet_vocab_workspace_bytes(p, D, M, V, D, 0, dtype, 0)
            assert lib.gnet_xent_forward(p, D, p, D, p, 1, M, V, D, dtype, p, p, p, p, need - 1, None) == _lib.ERR_WORKSPACE
            need = lib.gnet_vocab_workspace_bytes(p, D, M, V, D, 5, dtype, 1)
            assert lib.gnet_distill_backward(p, D, p, D, p, 0, p, 1.0, p, p, p, M, V, D, 5, dtype, p, p, p, need - 1, None) == _lib.ERR_WORKSPACE
    # (a small vocabulary: what its backward pass keeps fits into what is asked for)
    for M, V, D in ((1, 1, 1), (8192, 256, 16), (4097, 81, 128)):
        assert lib.gnet_vocab_workspace_bytes(p, D, M, V, D, 0, F32, 1) >= (M + 15) // 16 * 16 * ((V + 15) // 16 * 16 + 1) * 4
