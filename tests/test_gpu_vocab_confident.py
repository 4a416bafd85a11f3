"""Cross entropy's gradient in confident rows: the label's softmax is 1 but for 1e-7 to 1e-3, and the logits, and with them lse, are
hundreds.  With the forward's loss the gradient is off by the logits' errors and the sum's, not by lse's rounding.

Bounds (u = 2^-24), with r = 1 - softmax of the label:
  loss      the label's logit is the row's largest, from the same products: top - hit = 0.  The sum of exp(z - top) is 1 + r / (1 - r): its
            small terms are off as the logits are (2 max dz) and by 8 u of the difference and exp2, relative to r; the partial sum that holds the 1
            takes part in at most 64 additions (a lane's terms, the lanes, the waves, the tiles), each off by u, and log and expm1 are
            off by 8 u together: 72 u and 4 u of r.
  others    dz = p = exp(z - lse), off by p (dz + dl) as in test_gpu_vocab.py
  products  as there"""
import pytest
import torch

from test_gpu_vocab import DEV, TYPES, U, Exact, half_step, near, store_step

pytestmark = pytest.mark.gpu


def confident(M, V, D, dtype, seed, level=1000.0):
    """Logits `level` + a little, the label's 12 to 24 above the rest, so that 1 - softmax is 1e-7 to 1e-3."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[dtype]
    w = torch.randn(V, D, device=DEV, generator=g) * D ** -0.5
    w[:, 0] = 1.0
    labels = torch.randint(0, V, (M,), device=DEV, generator=g)
    above = 12 + 12 * torch.rand(M, 1, device=DEV, generator=g)
    own = w[labels].clone()
    own[:, 0] = 0
    x = own / own.pow(2).sum(1, keepdim=True) * above
    x[:, 0] = level
    return x.to(t), w.to(t), labels, torch.rand(M, device=DEV, generator=g) + 0.5


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,V,D", [(90, 700, 128), (600, 3000, 192), (200, 100, 1024), (150, 900, 2240), (20, 700, 128), (20, 700, 131), (90, 81, 128), (2000, 81, 64)])
def test_gradients_of_confident_rows(dtype, M, V, D):
    from gossipnet_amd import vocab
    x, w, labels, dloss = confident(M, V, D, dtype, M + V)
    e = Exact(x, w, labels)
    rows = torch.arange(M, device=DEV)
    z = e.x @ e.w.t()
    at = z[rows, labels]
    others = torch.exp(z - at[:, None])
    others[rows, labels] = 0
    s = others.sum(1)
    r = s / (1 + s)                                                    # 1 - softmax without a difference
    assert float(r.min()) < 1e-5 and float(r.max()) < 0.5
    off = 2 * e.dz_err.amax(1) + 8 * U
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    near(loss, torch.log1p(s), torch.log1p(s) * (off + 4 * U) + 72 * U, "loss")
    dx, dw = vocab.xent_backward(x, w, labels, lse, hit, dloss, loss=loss)
    g = dloss.double()[:, None]
    dz = others / (1 + s)[:, None]
    err = dz * (e.dz_err + e.lse_err[:, None] + 8 * U)
    dz[rows, labels] = -r
    err[rows, labels] = r * (off + 8 * U) + 72 * U
    dz, err = dz * g, err * g + store_step(e.t) * dz.abs() * g + 2.0 ** -38 * g.max()
    for got, a, b, q, n, what in ((dx, dz, e.w, err, V, "dx"), (dw, dz.t(), e.x, err.t(), M, "dw")):
        exact = a @ b
        tol = q @ b.abs() + (n + 8) * U * (a.abs() @ b.abs()) + half_step(e.t) * exact.abs() * (1 + 2.0 ** -6)
        if dtype == "f32":
            tol += 2.0 ** -38 * b.abs().max() * a.abs().sum(1, keepdim=True) + 2.0 ** -22 * (a.abs() @ b.abs())
        near(got, exact, tol, what)


def test_the_loss_is_checked_and_may_be_left_out():
    from gossipnet_amd import _lib, vocab
    x, w, labels, dloss = confident(40, 300, 64, "bf16", 5, 0.0)
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    with pytest.raises(_lib.InvalidArgumentError, match="loss has shape"):
        vocab.xent_backward(x, w, labels, lse, hit, dloss, loss=loss[1:])
    a, b = vocab.xent_backward(x, w, labels, lse, hit, dloss), vocab.xent_backward(x, w, labels, lse, hit, dloss, loss=loss)
    # away from the label nothing changes: dw of rows that are no token's label
    free = torch.ones(300, dtype=torch.bool, device=DEV)
    free[labels] = False
    assert torch.equal(a[1][free], b[1][free])
    labels[::3] = -1
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    dx, _ = vocab.xent_backward(x, w, labels, lse, hit, dloss, loss=loss)
    assert not bool(dx[::3].any()) and bool(dx[1].any())


def test_one_number_for_all_tokens():
    """A number in place of a tensor of the losses' gradients, eagerly and in a captured graph."""
    from gossipnet_amd import vocab
    x, w, labels, _ = confident(40, 300, 64, "bf16", 6, 0.0)
    ids, logits = torch.stack([labels, (labels + 1) % 300], 1), torch.randn(40, 2, device=DEV)
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    _, lse2, hit2 = vocab.distill_forward(x, w, ids, logits, 2.0)

    def both(g):
        return vocab.xent_backward(x, w, labels, lse, hit, g, loss=loss) + vocab.distill_backward(x, w, ids, logits, lse2, hit2, g, 2.0)
    want = both(torch.full((40,), 0.25, device=DEV))
    for g in (0.25, torch.tensor(0.25, device=DEV)):
        for a, b in zip(both(g), want):
            assert torch.equal(a, b)
    for a, b in zip(both(1), both(torch.ones(40, device=DEV))):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(0.25)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
