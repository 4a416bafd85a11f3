"""Tokens that are left out of the embedding's calls, whatever their rows and factors hold; the bounds are exact, the sums are of small whole
numbers."""
import math

import pytest
import torch

from test_gpu_vocab import DEV, TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,V,D", [(40, 3000, 72), (64, 40, 513), (1500, 30, 40), (5000, 7, 9), (5000, 100000, 8), (40000, 20, 33)])
def test_nothing_of_a_token_that_is_left_out_is_used(dtype, M, V, D):
    from gossipnet_amd import vocab
    t = TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(M + V)
    ids = torch.randint(0, V, (M,), device=DEV, generator=g)
    out = torch.rand(M, device=DEV, generator=g) < 0.3
    ids[out] = torch.tensor([-1, V, -2 ** 40, 2 ** 33], device=DEV)[torch.randint(0, 4, (int(out.sum()),), device=DEV, generator=g)]
    table = torch.randint(-2, 3, (V, D), device=DEV, generator=g).to(t)
    dy = torch.randint(-1, 2, (M, D), device=DEV, generator=g).to(t)
    s = torch.randint(1, 3, (M,), device=DEV, generator=g).float()
    clean = dy.clone()
    clean[out] = 0
    dy[out], s[out] = math.nan, math.inf
    ok = ~out
    y = vocab.embed_forward(ids, table, 1.0, s)
    want = torch.zeros(M, D, device=DEV, dtype=t)
    want[ok] = (table[ids[ok]].float() * s[ok, None]).to(t)
    assert torch.equal(y, want)
    dt, ds = vocab.embed_backward(ids, dy, table, 1.0, s, need_dscale=True)
    sums = torch.zeros(V, D, device=DEV, dtype=torch.float64).index_add_(0, ids[ok], dy[ok].double() * s[ok, None].double())
    assert torch.equal(dt, sums.to(t))
    dots = torch.zeros(M, device=DEV)
    dots[ok] = (table[ids[ok]].float() * dy[ok].float()).sum(1)
    assert torch.equal(ds, dots)
    acc = torch.ones(V, D, device=DEV, dtype=t)
    vocab.embed_backward(ids, dy, table, 1.0, s, out=acc)
    assert torch.equal(acc, (sums + 1).to(t))
