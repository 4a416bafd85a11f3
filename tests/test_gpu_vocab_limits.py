"""The vocabulary operators where a launch has more workgroups than one row of a grid, up to sizes whose threads would pass 2^32 in one.
The tokens repeat with a short period: every one is compared with the formulas of the first (the bounds of test_gpu_vocab.py)."""
import pytest
import torch

from test_gpu_vocab import DEV, TYPES, U, Exact, make, near

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def near_every_period(t, exact, tol, what):
    """(Not the same bits in each: a token whose tile of logits is worked on as two halves has the tile's sum put together from four
    waves' in place of two waves'.)"""
    t = t.reshape((-1,) + exact.shape)
    tol = torch.as_tensor(tol, device=t.device).expand_as(exact)
    for a in range(0, t.shape[0], 64):
        part = t[a:a + 64]
        near(part, exact.expand_as(part), tol.expand_as(part), what)


def check_periodic(x, w, ids, logits, tau, dloss, periods):
    """ids [n] or [n, K]; logits None: cross entropy."""
    from gossipnet_amd import vocab
    n = ids.shape[0]
    e = Exact(x, w, ids, logits, tau)
    X, I, G = x.repeat(periods, 1), ids.repeat((periods,) + (1,) * (ids.dim() - 1)), dloss.repeat(periods)
    if logits is None:
        loss, lse, hit = vocab.xent_forward(X, w, I)
        dx, dw = vocab.xent_backward(X, w, I, lse, hit, G)
        near_every_period(hit, e.hit[:, 0], e.hit_err[:, 0], "hit")
    else:
        T = logits.repeat(periods, 1)
        loss, lse, hit = vocab.distill_forward(X, w, I, T, tau)
        dx, dw = vocab.distill_backward(X, w, I, T, lse, hit, G, tau)
        near_every_period(hit, e.hit, e.hit_err, "hit")
    near_every_period(lse, e.lse, e.lse_err, "lse")
    near_every_period(loss, e.loss, e.loss_err, "loss")
    (ex, tx), (ew, tw) = e.gradients(dloss)
    near_every_period(dx, ex, tx, "dx")
    # the sum over all periods: each term off as in one period, and the longer sum's own rounding
    dz = ((e.p - e.target) * torch.where(e.some, dloss.double(), 0.0)[:, None] / tau).abs()
    near(dw, ew * periods, periods * (tw + (n * periods + 8) * U * (dz.t() @ e.x.abs())), "dw")


def test_slots_of_a_teacher_beyond_one_row_of_workgroups():
    """300 x 1024 tokens with 1024 slots: a wave for every four slots is 1.2 x 2^32 threads."""
    x, w, ids, dloss, logits = make(1024, 600, 64, "bf16", 1, 1024)
    ids[::4, 500:] = -1
    ids[5] = -1
    check_periodic(x, w, ids.int(), logits, 2.0, dloss, 300)


@pytest.mark.parametrize("dtype,M,V", [("bf16", 2 ** 21, 2 ** 18), ("f32", 2 ** 17, 2 ** 16)])
def test_many_tiles_of_logits(dtype, M, V):
    """2^39 logits of a width of 8: 2^23 tiles, in several launches."""
    n = 256
    x, w, labels, dloss = make(n, V, 8, dtype, 2)
    labels[::5] = -1
    check_periodic(x, w, labels, None, 1.0, dloss, M // n)


@pytest.mark.parametrize("M", [3, 64, 65, 3000])
def test_table_of_two_to_the_thirty_rows(M):
    from gossipnet_amd import vocab
    V = 2 ** 30
    g = torch.Generator(device=DEV).manual_seed(M)
    ids = torch.randint(0, V, (M,), device=DEV, generator=g)
    ids[0], ids[1], ids[2] = 0, V - 1, V
    dy = torch.randint(1, 9, (M, 1), device=DEV, generator=g).bfloat16()
    table = torch.empty(V, 1, device=DEV, dtype=torch.bfloat16)
    table[ids[ids < V]] = 2.0
    ok = ids < V
    y = vocab.embed_forward(ids, table)
    assert torch.equal(y[:, 0], torch.where(ok, 2.0, 0.0).bfloat16())
    dt, ds = vocab.embed_backward(ids, dy, table, need_dscale=True)
    want = torch.zeros(V, 1, device=DEV, dtype=torch.float32).index_add_(0, ids[ok], dy[ok].float()).bfloat16()
    assert torch.equal(dt, want)
    assert torch.equal(ds, torch.where(ok, 2.0 * dy[:, 0].float(), 0.0))
    vocab.embed_backward(ids, dy, table, out=dt)                    # rows without a token stay, also behind the last workgroup
    assert torch.equal(dt, (2 * want.float()).bfloat16())


@pytest.mark.parametrize("dtype,D", [("f32", 769), ("bf16", 1537)])
def test_rows_of_two_to_the_twenty_four_tokens(dtype, D):
    """Four waves a row, 2^32 threads: 52 GB of rows."""
    from gossipnet_amd import vocab
    M, V = 2 ** 24, 5
    g = torch.Generator(device=DEV).manual_seed(D)
    table = torch.randn(V, D, device=DEV, generator=g).to(TYPES[dtype])
    ids = torch.randint(0, V, (M,), device=DEV, generator=g, dtype=torch.int32)
    y = vocab.embed_forward(ids, table)
    for a in range(0, M, 2 ** 20):
        assert torch.equal(y[a:a + 2 ** 20], table[ids[a:a + 2 ** 20].long()])


@pytest.mark.parametrize("M,V,D", [(30, 5000, 96), (700, 90, 64), (5000, 3000, 72)])
def test_a_table_that_is_its_own_gradients_sum(M, V, D):
    """out=table: a step down the gradient in place."""
    from gossipnet_amd import vocab
    g = torch.Generator(device=DEV).manual_seed(M)
    table = torch.randint(-8, 9, (V, D), device=DEV, generator=g).float()
    ids = torch.randint(-1, V, (M,), device=DEV, generator=g)
    dy = torch.randint(-8, 9, (M, D), device=DEV, generator=g).float()
    want = table - 0.5 * vocab.embed_backward(ids, dy, table)[0]       # (sums of small multiples of a half: exact)
    assert vocab.embed_backward(ids, dy, table, -0.5, out=table)[0] is table
    assert torch.equal(table, want)
