"""The vocabulary operators at their limits, without a GPU: what is beyond is refused before anything is launched, what is within is taken."""
import ctypes as C
import random

import pytest

from gossipnet_amd import _lib

F32, BF16, F16 = 0, 1, 2
P = C.c_void_p(1 << 20)


def xent(M, V, D, dtype=BF16, backward=False, K=0):
    """Status of a call without a workspace: ERR_WORKSPACE where the sizes are taken."""
    lib = _lib.load()
    n = 0
    if K and backward:
        return lib.gnet_distill_backward(P, D, P, D, P, 0, P, 1.0, P, P, P, M, V, D, K, dtype, P, P, None, n, None)
    if K:
        return lib.gnet_distill_forward(P, D, P, D, P, 0, P, 1.0, M, V, D, K, dtype, P, P, P, None, n, None)
    if backward:
        return lib.gnet_xent_backward(P, D, P, D, P, 1, P, P, P, M, V, D, dtype, P, P, None, n, None)
    return lib.gnet_xent_forward(P, D, P, D, P, 1, M, V, D, dtype, P, P, P, None, n, None)


def embed(M, V, D, dtype=BF16):
    return _lib.load().gnet_embed_backward(P, 0, P, D, 1.0, None, M, V, D, dtype, P, 0, P, D, P, None, 0, None)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_matrices_beyond_the_limit_are_refused(dtype):
    """Fewer elements than 2^38 are what one launch can deal with; the sizes below pass every other limit."""
    lib = _lib.load()
    for backward in (False, True):
        for K in (0, 3):
            assert xent(1 << 24, 300, (1 << 14) + 1, dtype, backward, K) == _lib.ERR_UNSUPPORTED
            assert xent(300, 1 << 30, 257, dtype, backward, K) == _lib.ERR_UNSUPPORTED
            assert xent(1 << 24, 300, 1 << 14, dtype, backward, K) == _lib.ERR_WORKSPACE
            assert xent(300, 1 << 30, 256, dtype, backward, K) == _lib.ERR_WORKSPACE
    assert embed(1 << 24, 300, (1 << 14) + 1, dtype) == embed(300, 1 << 30, 257, dtype) == _lib.ERR_UNSUPPORTED
    assert embed(1 << 24, 300, 1 << 14, dtype) == embed(300, 1 << 30, 256, dtype) == _lib.ERR_WORKSPACE
    assert lib.gnet_embed_forward(P, 0, P, 1 << 16, 1.0, None, 1 << 24, 5, 1 << 16, dtype, P, None) == _lib.ERR_UNSUPPORTED


def test_what_is_within_the_limits_is_taken():
    """No size within the stated limits is refused for the size of a launch."""
    rng = random.Random(7)
    for n in range(4000):
        M, V, D = 1 << rng.randint(6, 24), 1 << rng.randint(9, 30), 1 << rng.randint(0, 16)
        if rng.random() < 0.7:
            M, V, D = max(65, M - rng.randint(0, M // 2)), max(300, V - rng.randint(0, V // 2)), max(1, D - rng.randint(0, D // 2))
        while M * V > 1 << 44:
            V = max(300, V >> 1)
            M = M >> 1 if V == 300 else M
        while max(M, V) * D > 1 << 38:
            D = max(1, D >> 1)
        case = (M, V, D, rng.choice([F32, BF16, F16]), rng.random() < 0.5, rng.choice([0, 1024]))
        assert xent(*case) == _lib.ERR_WORKSPACE, case


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [1 << 12, 1 << 17, 1 << 20, 1 << 24])
@pytest.mark.parametrize("V,D", [(50304, 1024), (50304, 64), (1 << 18, 8)])
def test_workspaces_grow_with_the_tokens_as_documented(M, V, D, dtype):
    """Copies of x, dx's fp32 sums and one piece of dz: 256 MB or 4 KB a token (fp32: 8 KB), and no more for a larger vocabulary but for W's copy."""
    planes = 2 if dtype == F32 else 1
    Mp, Dp = (M + 63) // 64 * 64, (D + 63) // 64 * 64
    lib = _lib.load()
    small = 64 * Mp + (1 << 20)                                        # per-token values
    copies = planes * planes * 2 * Mp * Dp                             # fp32: two copies of two planes
    sums = 16 * 4 * max(Mp * Dp, 512 * 256 * 256)                      # dx's sums, split at most 16 ways; dw's likewise in a small piece
    piece = max(256 << 20, planes * 2 * 2048 * (Mp + Dp) + (1 << 20))
    need = lib.gnet_vocab_workspace_bytes(P, D, M, V, D, 0, dtype, 1)
    assert need < small + copies + piece + (4 * Mp * Dp if M >= 1 << 17 else sums) + (256 << 20), need
    assert lib.gnet_vocab_workspace_bytes(P, D, M, 4 * V, D, 0, dtype, 1) <= need + (256 << 20)


def test_a_gradient_on_memory_that_is_read_is_refused():
    import torch
    from gossipnet_amd import vocab
    both = torch.zeros(30, 8)
    table, ids, dy = torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 8)
    for call in (lambda: vocab.embed_backward(ids, both[8:12], table, out=both[:10]),                  # dy begins inside out
                 lambda: vocab.embed_backward(ids, both[:4], table, out=both[3:13]),
                 lambda: vocab.embed_backward(ids, dy, table, need_dscale=True, out=table),
                 lambda: vocab.embed_backward(ids, dy, both[9:19], need_dscale=True, out=both[:10])):
        with pytest.raises(_lib.InvalidArgumentError, match="shares memory"):
            call()
    for call in (lambda: vocab.embed_backward(ids, both[10:14], table, out=both[:10]),                 # side by side
                 lambda: vocab.embed_backward(ids, both[:4], table, out=both[4:14]),
                 lambda: vocab.embed_backward(ids, dy, table, -0.1, out=table),                        # table is not read
                 lambda: vocab.embed_backward(ids[:0], dy[:0], table, out=table)):
        with pytest.raises(_lib.GnetError, match="device kernels"):
            call()


def test_a_number_is_taken_as_the_losses_gradient():
    import torch
    from gossipnet_amd import vocab
    x, w, y, one = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    for g in (1.0, 1, torch.tensor(1.0)):                              # (as far as the check of the device)
        with pytest.raises(_lib.GnetError, match="device kernels"):
            vocab.xent_backward(x, w, y, one, one, g)
        with pytest.raises(_lib.GnetError, match="device kernels"):
            vocab.distill_backward(x, w, y[:, None], one[:, None], one, one[:, None], g)


def test_the_entry_with_the_loss_refuses_like_the_one_without():
    lib = _lib.load()
    odd = C.c_void_p((1 << 20) + 8)

    def back(x=P, ldx=8, w=P, ldw=8, y=P, loss=P, lse=P, hit=P, g=P, M=65, V=3000, D=8, dtype=F32, ws=P, n=1 << 40):
        return lib.gnet_xent_backward_loss(x, ldx, w, ldw, y, 1, loss, lse, hit, g, M, V, D, dtype, P, P, ws, n, None)
    for a in (dict(M=-1), dict(V=0), dict(D=0), dict(ldx=7), dict(ldw=7), dict(dtype=3), dict(x=None), dict(w=None), dict(y=None), dict(lse=None), dict(hit=None), dict(g=None)):
        assert back(**a) == _lib.ERR_INVALID, a
    for a in (dict(M=(1 << 24) + 1), dict(V=(1 << 30) + 1), dict(D=(1 << 16) + 1, ldx=1 << 17, ldw=1 << 17)):
        assert back(**a) == _lib.ERR_UNSUPPORTED, a
    for V in (10, 3000):
        for M in (20, 65):
            need = lib.gnet_vocab_workspace_bytes(P, 8, M, V, 8, 0, F32, 1)
            for loss in (P, None):
                for a in (dict(ws=None), dict(n=need - 1), dict(ws=odd)):
                    assert back(M=M, V=V, loss=loss, **a) == _lib.ERR_WORKSPACE, a
