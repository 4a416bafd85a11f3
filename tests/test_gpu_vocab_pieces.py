"""The vocabulary losses where the vocabulary is worked on in several pieces, with W read in place and laid out, both losses and both directions
(the bounds of test_gpu_vocab.py).

A piece's dz and laid-out rows of W (planes x 2 bytes x (tokens and width, each up to 64) a row) take 256 MB at most; that there is more
than one is read off the workspace, which one piece for all rows would not fit into."""
import ctypes as C

import pytest
import torch

from test_gpu_vocab import DEV, check_distill, check_xent, make

pytestmark = pytest.mark.gpu

# type, tokens, vocabulary, width, W is laid out
CASES = [("f32", 300, 40000, 4096, True), ("bf16", 300, 70000, 4095, True), ("f16", 40, 70001, 4090, True), ("bf16", 4100, 70000, 64, False),
         ("f16", 2500, 120000, 72, False), ("f32", 2050, 70001, 61, True), ("f32", 40, 33000, 8200, True)]


def more_than_one_piece(dtype, M, V, D, K, laid_out):
    from gossipnet_amd import _lib
    planes = 2 if dtype == "f32" else 1
    up = lambda n: (n + 63) // 64 * 64                                 # noqa: E731
    w = C.c_void_p(1 << 20)
    code = {"f32": 0, "bf16": 1, "f16": 2}[dtype]
    back = _lib.load().gnet_vocab_workspace_bytes(w, D, M, V, D, K, code, 1)
    ahead = _lib.load().gnet_vocab_workspace_bytes(w, D, M, V, D, K, code, 0)
    rows = planes * 2 * V
    assert back < rows * (up(M) + (up(D) if laid_out else 0)), (back, rows)
    return ahead < rows * up(D) and laid_out                           # and in the forward pass?


@pytest.mark.parametrize("dtype,M,V,D,laid_out", CASES)
def test_xent_in_pieces(dtype, M, V, D, laid_out):
    assert more_than_one_piece(dtype, M, V, D, 0, laid_out) == (laid_out and D > 2000)
    x, w, labels, dloss = make(M, V, D, dtype, 41)
    labels[::7] = -1
    labels[1], labels[2] = 0, V - 1                                    # the first row and the last
    check_xent(x, w, labels, dloss)


@pytest.mark.parametrize("dtype,M,V,D,laid_out", CASES[:5])
def test_distill_in_pieces(dtype, M, V, D, laid_out):
    more_than_one_piece(dtype, M, V, D, 5, laid_out)
    x, w, ids, dloss, logits = make(M, V, D, dtype, 42, 5)
    ids[::7] = -1
    ids[1] = torch.tensor([0, V - 1, V // 2, 0, V - 1], device=DEV)
    ids[2::5, 1] = V + 1
    check_distill(x, w, ids, logits, 1.5, dloss)


def test_a_step_in_pieces_captured_and_replayed():
    """Both losses over the same rows, gradients added, replayed with other inputs between eager calls."""
    from gossipnet_amd import vocab
    dtype, M, V, D, laid_out = CASES[1]
    assert more_than_one_piece(dtype, M, V, D, 0, laid_out)
    x, w, ids, dloss, logits = make(M, V, D, dtype, 43, 3)
    labels = ids[:, 0].contiguous()

    def step():
        loss, lse, hit = vocab.xent_forward(x, w, labels)
        dx, dw = vocab.xent_backward(x, w, labels, lse, hit, dloss, loss=loss)
        loss2, lse, hit = vocab.distill_forward(x, w, ids, logits, 2.0)
        dx2, dw2 = vocab.distill_backward(x, w, ids, logits, lse, hit, dloss, 2.0)
        return loss, loss2, dx + dx2, dw + dw2
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        x.copy_(torch.randn(M, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(turn)))
        labels.copy_(labels.roll(turn + 1))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), turn
