"""The vocabulary losses on operands and gradients far from 1: what scales the matrix products' operands has to cancel for every magnitude
(the bounds of test_gpu_vocab.py)."""
import pytest
import torch

from test_gpu_vocab import DEV, Exact, check_distill, check_xent, make, near

pytestmark = pytest.mark.gpu

# (tokens, vocabulary, width) of: tiles of logits, a vocabulary of one tile, a contraction in parts, few tokens, a small vocabulary
PATHS = [(90, 700, 128), (90, 100, 1024), (150, 900, 2240), (20, 700, 128), (90, 81, 128)]


@pytest.mark.parametrize("M,V,D", PATHS)
def test_operands_whose_scales_multiply_to_less_than_a_float_holds(M, V, D):
    """x and w around 1e-20 and below: the logits are 0, lse = log V, and no row behind the last one takes part."""
    x, w, labels, dloss = make(M, V, D, "f32", 21)
    for a, b in ((1e-20, 1e-20), (1e-30, 1e-12), (1e-12, 1e-30)):
        e = check_xent(x * a, w * b, labels, dloss)
        assert bool(((e.lse - float(torch.tensor(float(V)).log())).abs() < 1e-5).all())
    x, w, ids, dloss, logits = make(M, V, D, "f32", 22, 3)
    check_distill(x * 1e-20, w * 1e-20, ids, logits, 2.0, dloss)


@pytest.mark.parametrize("M,V,D", PATHS)
def test_a_zero_row_beside_the_largest_values(M, V, D):
    """x and w around 1e37: other tokens' logits are infinite, a token of zeros has logits 0."""
    from gossipnet_amd import vocab
    x, w, labels, dloss = make(M, V, D, "f32", 23)
    x, w = x.clamp(-4, 4) * 1e37, w.clamp(-4, 4) * 1e37
    x[3] = 0
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    e = Exact(torch.zeros(1, D, device=DEV), w, labels[3:4])
    assert abs(float(lse[3]) - float(e.lse[0])) < 1e-5 and abs(float(loss[3]) - float(e.lse[0])) < 1e-5 and float(hit[3]) == 0


@pytest.mark.parametrize("M,V,D", PATHS)
@pytest.mark.parametrize("sx,sw,sg", [(2.0 ** -50, 1.0, 2.0 ** -66), (1.0, 2.0 ** -50, 2.0 ** -66), (2.0 ** -40, 2.0 ** 40, 2.0 ** -75), (2.0 ** 60, 2.0 ** -60, 2.0 ** 60),
                                      (2.0 ** -60, 2.0 ** 60, 2.0 ** 60)])
def test_small_and_large_gradients_of_small_and_large_operands(M, V, D, sx, sw, sg):
    """Powers of two on x, w and the losses' gradient: dx and dw as far off as without them (and as the bounds say), relative to their own size."""
    from gossipnet_amd import vocab
    x, w, labels, dloss = make(M, V, D, "f32", 24)
    x, w, dloss = x * sx, w * sw, dloss * sg
    e = Exact(x, w, labels)
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    for got, (exact, tol), size in zip(vocab.xent_backward(x, w, labels, lse, hit, dloss), e.gradients(dloss), (sw * sg, sx * sg)):
        near(got.double() / size, exact / size, tol / size, "gradient")


@pytest.mark.parametrize("M,V,D", PATHS)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_an_infinity_stays_with_its_token(dtype, M, V, D):
    """A token that counts, with an infinity in its row or in its loss' gradient: every other token's results are what they are without it."""
    from gossipnet_amd import vocab
    x, w, labels, dloss = make(M, V, D, dtype, 25)
    if dtype == "f32":
        x, w = x * 1e6, w * 1e-6                                       # beyond what 16 bits hold without a scale
    dloss = dloss.sign() * 5.0
    others = torch.arange(M, device=DEV) != 7
    e = Exact(x, w, labels)
    want = vocab.xent_forward(x, w, labels)
    g = torch.where(others, dloss, float("inf"))
    dx, _ = vocab.xent_backward(x, w, labels, want[1], want[2], g)
    exact, tol = e.gradients(dloss)[0]
    near(dx[others], exact[others], tol[others], "dx")
    assert not bool(dx[7].isfinite().any())
    bad = x.clone()
    bad[7, 3] = float("inf")
    loss, lse, hit = vocab.xent_forward(bad, w, labels)
    near(hit[others], e.hit[others, 0], e.hit_err[others, 0], "hit")
    near(lse[others], e.lse[others], e.lse_err[others], "lse")
    near(loss[others], e.loss[others], e.loss_err[others], "loss")
    assert not bool(loss[7].isfinite())
    dx, _ = vocab.xent_backward(bad, w, labels, lse, hit, dloss)
    near(dx[others], exact[others], tol[others], "dx")
    assert not bool(dx[7].isfinite().any())
