"""Losses weighted very differently within one call: every token's dx has the accuracy of its own weight.

The bound of a row of dx is that of test_gpu_vocab.py with the row's own gradient in place of the largest: two fp16 hold dz of a token
to 2^-22 of itself and 2^-38 of the token's |dloss|.  fp16 operands hold dz in one fp16 in units of the largest |dloss| / 2^15: half a step of itself, and at
the lower end 2^-25 of that unit, 2^-40 of the largest.  bf16 has fp32's range: half a step."""
import pytest
import torch

from test_gpu_vocab import DEV, U, Exact, half_step, make, near, store_step

pytestmark = pytest.mark.gpu


def rows_of_dx(e, dloss):
    """dx and its bound, row by row."""
    g = torch.where(e.some, dloss.double(), 0.0)[:, None] / e.tau
    dz = (e.p - e.target) * g
    err = g.abs() * e.p * (e.dz_err + e.lse_err[:, None] + 8 * U) + store_step(e.t) * dz.abs()
    if e.t == torch.float32:
        err += 2.0 ** -38 * g.abs()
    if e.t == torch.float16:
        err += 2.0 ** -40 * g.abs().max()
    err += g.abs() * e.target * (16 * U if e.target.max() < 1 or e.tau != 1 else 2 * U)
    a, b = dz, e.w
    exact = a @ b
    tol = err @ b.abs() + (e.V + 8) * U * (a.abs() @ b.abs()) + half_step(e.t) * exact.abs() * (1 + 2.0 ** -6)
    if e.t == torch.float16:
        tol += 2.0 ** -25
    if e.t == torch.float32:
        tol += 2.0 ** -38 * b.abs().max() * a.abs().sum(1, keepdim=True) + 2.0 ** -22 * (a.abs() @ b.abs())
    return exact, tol


@pytest.mark.parametrize("M,V,D", [(90, 700, 128), (300, 2000, 192), (90, 100, 1024), (150, 900, 2240), (500, 30000, 256), (20, 700, 131), (90, 81, 128)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("least", [1e-10, 1e-25])
def test_weights_of_many_magnitudes(M, V, D, dtype, least):
    from gossipnet_amd import vocab
    x, w, labels, dloss = make(M, V, D, dtype, 31)
    g = torch.Generator(device=DEV).manual_seed(M)
    weight = least ** torch.rand(M, device=DEV, generator=g)
    dloss = dloss.sign() * weight
    dloss[3] = 0
    labels[::7] = -1
    e = Exact(x, w, labels)
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    dx, dw = vocab.xent_backward(x, w, labels, lse, hit, dloss)
    exact, tol = rows_of_dx(e, dloss)
    size = weight.double()[:, None] if dtype != "f16" else 1.0         # (results in fp16 have steps of 2^-24)
    near(dx.double() / size, exact / size, tol / size, "dx")
    (_, _), (ew, tw) = e.gradients(dloss)
    near(dw, ew, tw, "dw")
    ids, logits = make(M, V, D, dtype, 32, 4)[2], make(M, V, D, dtype, 32, 4)[4]
    e = Exact(x, w, ids, logits, 2.0)
    loss, lse, hit = vocab.distill_forward(x, w, ids, logits, 2.0)
    dx, dw = vocab.distill_backward(x, w, ids, logits, lse, hit, dloss, 2.0)
    exact, tol = rows_of_dx(e, dloss)
    near(dx.double() / size, exact / size, tol / size, "dx")
    (_, _), (ew, tw) = e.gradients(dloss)
    near(dw, ew, tw, "dw")
