"""The vocabulary operators against their formulas in 64 bits.

Tolerances follow from the arithmetic, element by element (u = 2^-24, h = half a step of the type: finfo.eps / 2):
  logits      products of 16-bit inputs are exact; a sum of D terms in fp32 is off by at most D u sum|x w|; the two fp16 of an fp32
              operand and the dropped lo.lo add 3 x 2^-24 of sum|x w| (and 2^-38 of the tensors' largest magnitudes):
              dz = (D + 8) u sum|x w| / temperature + 2 u |z|
  lse         the logits' errors, and a sum of positive terms over a tree of at most 2 x 64 levels, exp2 and log2 to an ulp or two
              each, in units of log2:  dl = max dz + 160 u + 4 u |lse|
  dz matrix   p = exp(z - lse) is off by p (dz + dl + 8 u); stored with half a step: h for 16 bits, 2^-22 for the two fp16, which end
              at 2^-38 of the largest |dloss|
  products    a sum of n terms in fp32: n u of the sum of magnitudes; the result's rounding h."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def store_step(t):
    return 2.0 ** -22 if t == torch.float32 else half_step(t)


def make(M, V, D, dtype, seed, K=None, spread=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[dtype]
    w = (torch.randn(V, D, device=DEV, generator=g) * (spread * D ** -0.5)).to(t)
    x = torch.randn(M, D, device=DEV, generator=g)
    ids = torch.randint(0, V, (M,) if K is None else (M, K), device=DEV, generator=g)
    x += 3.0 * w[ids if K is None else ids[:, 0]].float()
    out = [x.to(t), w, ids, torch.randn(M, device=DEV, generator=g) / M]
    if K is not None:
        out.append(torch.randn(M, K, device=DEV, generator=g) * 2 + 5)
    return out


class Exact(object):
    """The formulas in 64 bits, with the bounds of the header (ids [M,K], logits [M,K] or None: one target of weight 1)."""

    def __init__(self, x, w, ids, logits=None, temperature=1.0):
        M, V = ids.shape[0], w.shape[0]
        ids = ids.long().reshape(M, -1)
        ok = (ids >= 0) & (ids < V)
        self.t, self.tau, self.V, self.D = x.dtype, temperature, V, x.shape[1]
        if logits is not None:
            ok &= logits != -math.inf
        self.some = some = ok.any(1)
        self.x = torch.where(some[:, None], x.double(), 0.0)          # rows that are left out may hold anything
        self.w = w.double()
        z = self.x @ self.w.t() / temperature
        self.mag = self.x.abs() @ self.w.abs().t() / temperature
        self.lse = torch.where(some, torch.logsumexp(z, 1), 0.0)
        tz = torch.zeros_like(ids, dtype=torch.float64) if logits is None else logits.double() / temperature
        tz = tz.masked_fill(~ok, -math.inf)
        logq = torch.where(some[:, None], torch.log_softmax(tz, 1), -math.inf)
        self.q = q = logq.exp()
        idc = ids.clamp(0, V - 1)
        self.hit = torch.where(ok, z.gather(1, idc), 0.0)
        self.loss = torch.where(ok & (q > 0), q * (logq - self.hit + self.lse[:, None]), 0.0).sum(1)
        self.dz_err = (self.D + 8) * U * self.mag + 2 * U * z.abs() + 2.0 ** -38 * self.x.abs().max() * self.w.abs().max() * self.D / temperature
        self.hit_err = torch.where(ok, self.dz_err.gather(1, idc), 0.0)
        self.lse_err = torch.where(some, self.dz_err.amax(1) + 160 * U + 4 * U * self.lse.abs(), 0.0)
        self.entropy_err = 0.0 if logits is None else 64 * U * (1 + torch.where(q > 0, logq, 0.0).abs().amax(1) + (tz.masked_fill(~ok, 0).abs().amax(1)))
        self.loss_err = self.lse_err + self.hit_err.amax(1) + 8 * U * (self.lse.abs() + self.hit.abs().amax(1)) + self.entropy_err
        self.p = torch.where(some[:, None], torch.exp(z - self.lse[:, None]), 0.0)
        self.target = torch.zeros_like(z)
        self.target.scatter_add_(1, idc, torch.where(ok, q, 0.0))

    def gradients(self, dloss):
        g = torch.where(self.some, dloss.double(), 0.0)[:, None] / self.tau
        dz = (self.p - self.target) * g
        err = g.abs() * self.p * (self.dz_err + self.lse_err[:, None] + 8 * U) + store_step(self.t) * dz.abs() + 2.0 ** -38 * g.abs().max()
        # the targets' weights: a softmax in fp32
        err += g.abs() * self.target * (16 * U if self.target.max() < 1 or self.tau != 1 else 2 * U)
        out = []
        for a, e, b, n in ((dz, err, self.w, self.V), (dz.t(), err.t(), self.x, dz.shape[0])):
            exact = a @ b
            tol = e @ b.abs() + (n + 8) * U * (a.abs() @ b.abs()) + half_step(self.t) * exact.abs() * (1 + 2.0 ** -6)
            if self.t == torch.float16:
                tol += 2.0 ** -25                  # a subnormal result's step
            if self.t == torch.float32:
                tol += 2.0 ** -38 * b.abs().max() * a.abs().sum(1, keepdim=True) + 2.0 ** -22 * (a.abs() @ b.abs())
            out.append((exact, tol))
        return out


def near(got, exact, tol, what):
    assert got.shape == exact.shape, what
    bad = ~((got.double() - exact).abs() <= tol + 1e-30)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.flatten())[0])
        tol = tol + torch.zeros_like(exact)
        raise AssertionError("%s: %d of %d beyond the bound, first at %d: %r against %r, bound %r"
                             % (what, int(bad.sum()), bad.numel(), i, float(got.flatten()[i]), float(exact.flatten()[i]), float(tol.flatten()[i])))


def check_xent(x, w, labels, dloss, back=True):
    from gossipnet_amd import vocab
    e = Exact(x, w, labels)
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    near(hit, e.hit[:, 0], e.hit_err[:, 0], "hit")
    near(lse, e.lse, e.lse_err, "lse")
    near(loss, e.loss, e.loss_err, "loss")
    if back:
        dx, dw = vocab.xent_backward(x, w, labels, lse, hit, dloss)
        assert dx.dtype == x.dtype and dw.dtype == w.dtype
        (ex, tx), (ew, tw) = e.gradients(dloss)
        near(dx, ex, tx, "dx")
        near(dw, ew, tw, "dw")
        assert not bool(dx[~e.some].any())
    return e


def check_distill(x, w, ids, logits, tau, dloss):
    from gossipnet_amd import vocab
    e = Exact(x, w, ids, logits, tau)
    loss, lse, hit = vocab.distill_forward(x, w, ids, logits, tau)
    near(hit, e.hit, e.hit_err, "hit")
    near(lse, e.lse, e.lse_err, "lse")
    near(loss, e.loss, e.loss_err, "loss")
    dx, dw = vocab.distill_backward(x, w, ids, logits, lse, hit, dloss, tau)
    (ex, tx), (ew, tw) = e.gradients(dloss)
    near(dx, ex, tx, "dx")
    near(dw, ew, tw, "dw")
    return e


SIZES = [(1, 1, 1), (1, 2, 3), (3, 5, 7), (2, 300, 64), (17, 130, 65), (64, 127, 64), (128, 128, 128), (129, 257, 192), (65, 1000, 100),
         (300, 513, 256), (5, 8191, 72), (31, 4099, 320), (513, 81, 128), (1100, 1030, 136), (3, 200, 8200), (9001, 130, 64), (270000, 40, 8),
         (165, 2283, 2240), (5, 154, 2050), (300, 129, 1100),
         (20, 120, 600), (50, 100, 700), (9000, 81, 128), (33, 256, 128), (17, 255, 129), (2000, 81, 128), (8192, 9, 30),
         (5, 3001, 129), (16, 1000, 592), (17, 700, 301), (32, 5000, 75), (32, 2049, 515), (33, 2049, 515), (20, 129, 1000), (16, 2048, 1024), (17, 2048, 1024), (2, 5000, 1032)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,V,D", SIZES)
def test_xent(M, V, D, dtype):
    x, w, labels, dloss = make(M, V, D, dtype, M + V + D)
    check_xent(x, w, labels, dloss)
    labels = labels.int()
    labels[::3] = -100
    check_xent(x, w, labels, dloss)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,V,D,K,tau", [(1, 1, 1, 1, 1.0), (1, 70, 64, 70, 2.0), (3, 5, 7, 2, 0.5), (17, 130, 65, 3, 4.0), (64, 500, 128, 64, 1.5), (200, 1111, 72, 65, 1.0),
                                         (40, 1000, 4100, 13, 2.5), (130, 300, 256, 8, 2.0), (5, 5000, 96, 200, 3.0), (3, 3000, 64, 1024, 2.0), (9001, 100, 64, 3, 1.0),
                                         (30, 200, 64, 64, 1.5), (517, 81, 100, 33, 2.0),
                                         (20, 700, 131, 9, 2.0), (32, 129, 777, 5, 1.0)])
def test_distill(M, V, D, K, tau, dtype):
    x, w, ids, dloss, logits = make(M, V, D, dtype, M + V + K, K)
    check_distill(x, w, ids, logits, tau, dloss)                       # random ids: some occur twice in a row
    ids = ids.int()
    ids[::4] = -1                                                      # tokens without a teacher
    ids[1::4, K // 2:] = V + 3                                         # fewer than K
    logits[2::4, ::2] = -math.inf
    check_distill(x, w, ids, logits, tau, dloss)


@pytest.mark.parametrize("V", [200, 700])
def test_same_id_in_every_slot_and_lowest_logits(V):
    x, w, ids, dloss, logits = make(40, V, 64, "bf16", 5, 6)
    ids[:] = ids[:, :1]
    check_distill(x, w, ids, logits, 2.0, dloss)
    ids = torch.arange(6, device=DEV).repeat(40, 1) * 30
    low = torch.finfo(torch.float32).min
    logits[::2, 1:] = low                                              # the type's lowest value weighs nothing beside others ...
    logits[1::4] = low                                                 # ... and as much as they do among its like
    check_distill(x, w, ids, logits, 1.0, dloss)
    logits[:] = -math.inf
    e = check_distill(x, w, ids, logits, 1.0, dloss)
    assert not bool(e.some.any())


@pytest.mark.parametrize("D", [64, 1000])
def test_labels_outside_the_vocabulary(D):
    from gossipnet_amd import vocab
    x, w, labels, dloss = make(9, 50, D, "bf16", 3)
    labels[:] = torch.tensor([-1, 50, -100, 2 ** 32 + 1, -2 ** 40, 51, 2 ** 31, 7, 2 ** 62], device=DEV)
    e = check_xent(x, w, labels, dloss)
    assert e.some.tolist() == [False] * 7 + [True, False]
    labels[7] = -5
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    dx, dw = vocab.xent_backward(x, w, labels, lse, hit, dloss)
    for t in (loss, lse, hit, dx, dw):
        assert not bool(t.any())


@pytest.mark.parametrize("M,V,D", [(150, 120, 128), (150, 333, 128), (20, 333, 131), (9, 900, 129)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_infinities_and_nan_in_rows_that_are_left_out(dtype, M, V, D):
    x, w, labels, dloss = make(M, V, D, dtype, 8)
    x[3], x[M // 2], x[M - 1] = math.nan, math.inf, -math.inf
    labels[3] = labels[M // 2] = labels[M - 1] = -1
    dloss[3], dloss[M // 2] = math.nan, math.inf
    check_xent(x, w, labels, torch.where(labels < 0, 0, dloss))
    check_xent(x, w, labels, dloss)


@pytest.mark.parametrize("V", [90, 700])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_logits_and_confident_rows(dtype, V):
    x, w, labels, dloss = make(100, V, 192, dtype, 9)
    check_xent(x * 300, w, labels, dloss)                              # far beyond exp's range
    check_xent(w[labels] * 40, w, labels, dloss)                       # the label takes nearly everything
    check_xent(x * 0, w, labels, dloss)                                # uniform


@pytest.mark.parametrize("V", [200, 600])
def test_outliers_in_fp32(V):
    """One power of two scales a whole tensor: rows and single values far above and far below the rest."""
    x, w, labels, dloss = make(90, V, 128, "f32", 16)
    x[5, 3], x[6] = 3e4, x[6] * 1e-6
    w[7], w[8], w[9, 1] = w[7] * 1e-8, w[8] * 50, 2000.0
    check_xent(x, w, labels, dloss)
    check_xent(x * 1e-20, w * 1e-15, labels, dloss)
    check_xent(x * 1e12, w * 1e-12, labels, dloss * 1e9)


@pytest.mark.parametrize("V", [100, 300])
def test_loss_gradients_of_all_sizes(V):
    x, w, labels, dloss = make(64, V, 128, "f16", 10)
    for scale in (1e-30, 1e-3, 1e4, 0.0):
        from gossipnet_amd import vocab
        e = Exact(x, w, labels)
        _, lse, hit = vocab.xent_forward(x, w, labels)
        g = dloss * scale
        dx, dw = vocab.xent_backward(x, w, labels, lse, hit, g)
        (ex, tx), (ew, tw) = e.gradients(g)
        near(dx, ex, tx, "dx")
        near(dw, ew, tw, "dw")
    # one number for all tokens; what is not needed is left out
    a = vocab.xent_backward(x, w, labels, lse, hit, torch.tensor(0.25, device=DEV))
    b = vocab.xent_backward(x, w, labels, lse, hit, torch.full((64,), 0.25, device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert vocab.xent_backward(x, w, labels, lse, hit, g, need_dx=False)[0] is None
    dx, dw = vocab.xent_backward(x, w, labels, lse, hit, torch.tensor(0.25, device=DEV), need_dw=False)
    assert dw is None and torch.equal(dx, a[0])


@pytest.mark.parametrize("dtype,M,V", [("f32", 70, 100), ("f32", 70, 260), ("f32", 70, 700), ("f32", 30, 700), ("bf16", 70, 100), ("bf16", 70, 260), ("bf16", 70, 700)])
def test_strides_and_alignment(dtype, M, V):
    """Rows inside wider ones, addresses that are no multiple of 16, transposed and expanded tensors: the dense call's results."""
    from gossipnet_amd import vocab
    D = 128
    x, w, labels, dloss = make(M, V, D, dtype, 11)

    def run(x, w):
        loss, lse, hit = vocab.xent_forward(x, w, labels)
        return (loss, lse, hit) + vocab.xent_backward(x, w, labels, lse, hit, dloss)
    want = run(x, w)
    for off, wide in ((0, 192), (1, 131), (8, 136), (3, 160)):
        bx, bw = torch.full((M, wide), 7.0, device=DEV, dtype=x.dtype), torch.full((V, wide), 7.0, device=DEV, dtype=x.dtype)
        bx[:, off:off + D], bw[:, off:off + D] = x, w
        for a, b in zip(want, run(bx[:, off:off + D], bw[:, off:off + D])):
            assert torch.equal(a, b)
    for a, b in zip(want, run(x.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(a, b)
    got = run(x[:1].expand(M, D), w)
    check_xent(x[:1].expand(M, D), w, labels, dloss)
    assert got[3].shape == (M, D)
    # leading dimensions
    y = labels.reshape(M // 10, 10)
    loss, lse, hit = vocab.xent_forward(x.reshape(M // 10, 10, D), w, y)
    dx, dw = vocab.xent_backward(x.reshape(M // 10, 10, D), w, y, lse, hit, dloss.reshape(M // 10, 10))
    assert torch.equal(loss.flatten(), want[0]) and torch.equal(dx.reshape(M, D), want[3]) and torch.equal(dw, want[4])


def test_one_token_without_dimensions():
    from gossipnet_amd import vocab
    x, w, labels, _ = make(1, 90, 64, "bf16", 15)
    one = torch.tensor(1.0, device=DEV)
    loss, lse, hit = vocab.xent_forward(x[0], w, labels[0])
    dx, dw = vocab.xent_backward(x[0], w, labels[0], lse, hit, one)
    a = vocab.xent_forward(x, w, labels)
    b = vocab.xent_backward(x, w, labels, a[1], a[2], one)
    assert loss.shape == lse.shape == hit.shape == () and float(loss) == float(a[0]) and dx.shape == (64,)
    assert torch.equal(dx, b[0][0]) and torch.equal(dw, b[1])
    y = vocab.embed_forward(labels[0], w)
    assert y.shape == (64,) and torch.equal(y, w[labels[0]])
    dt, ds = vocab.embed_backward(labels[0], y, w, need_dscale=True)
    assert ds.shape == () and torch.equal(dt[labels[0]], y)


def test_no_tokens():
    from gossipnet_amd import vocab
    for t in TYPES.values():
        w, x, y = torch.ones(5, 3, device=DEV, dtype=t), torch.ones(0, 3, device=DEV, dtype=t), torch.ones(0, device=DEV, dtype=torch.int64)
        loss, lse, hit = vocab.xent_forward(x, w, y)
        dx, dw = vocab.xent_backward(x, w, y, lse, hit, loss)
        assert loss.shape == (0,) and dx.shape == (0, 3) and dw.shape == (5, 3) and not bool(dw.any())
        e = vocab.embed_forward(y, w)
        assert e.shape == (0, 3)
        dt, ds = vocab.embed_backward(y, e, w, need_dscale=True)
        assert dt.shape == (5, 3) and not bool(dt.any()) and ds.shape == (0,)
        keep = torch.ones(5, 3, device=DEV, dtype=t)
        assert vocab.embed_backward(y, e, w, out=keep)[0] is keep and bool((keep == 1).all())


@pytest.mark.parametrize("dtype,M,V,D", [("bf16", 4100, 20011, 64), ("f32", 2050, 20011, 64), ("f16", 130, 3000, 2056)])
def test_several_pieces_of_the_vocabulary(dtype, M, V, D):
    x, w, labels, dloss = make(M, V, D, dtype, 12)
    labels[::7] = -1
    check_xent(x, w, labels, dloss)


def test_two_calls_at_once():
    """Two streams with calls of different shapes in flight: each gives what it gives alone."""
    from gossipnet_amd import vocab
    a, b = make(900, 20000, 512, "bf16", 30), make(300, 6000, 256, "f32", 31)

    def run(x, w, labels, dloss):
        loss, lse, hit = vocab.xent_forward(x, w, labels)
        return (loss, lse, hit) + vocab.xent_backward(x, w, labels, lse, hit, dloss) + (vocab.embed_backward(labels, x, w)[0],)
    want = [run(*a), run(*b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for k, (s, args) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[k].append(run(*args))
    torch.cuda.synchronize()
    for k in (0, 1):
        for out in got[k]:
            for p, q in zip(out, want[k]):
                assert torch.equal(p, q)


def test_repeats_are_bitwise_equal():
    from gossipnet_amd import vocab
    x, w, ids, dloss, logits = make(700, 3001, 512, "bf16", 13, 5)

    def run():
        loss, lse, hit = vocab.distill_forward(x, w, ids, logits, 2.0)
        out = (loss, lse, hit) + vocab.distill_backward(x, w, ids, logits, lse, hit, dloss, 2.0)
        e = vocab.embed_backward(ids, w[ids.clamp(0, 9)], w)[0]
        return out + (e,)
    a = run()
    for _ in range(3):
        for p, q in zip(a, run()):
            assert torch.equal(p, q)


def test_gradient_against_differences():
    """(L(x + s v) - L(x - s v)) / 2s against <dx, v> and the same for w, in fp32.  Both L are off by loss_err; the remainder of the
    difference quotient is at most s^2 / 6 of L's third derivative along v, which for a softmax of logits that move at rates r is below
    (max r - min r)^3 / 2 (a third central moment of a variable within that range is below range^3 / 10; w's part is linear in w)."""
    from gossipnet_amd import vocab
    x, w, labels, _ = make(6, 23, 64, "f32", 14)
    g = torch.Generator(device=DEV).manual_seed(1)
    ones = torch.ones(6, device=DEV)
    e = Exact(x, w, labels)
    loss, lse, hit = vocab.xent_forward(x, w, labels)
    dx, dw = vocab.xent_backward(x, w, labels, lse, hit, ones)
    for which, grad in (("x", dx), ("w", dw)):
        v = torch.randn(grad.shape, device=DEV, generator=g) * 0.3
        rate = (v.double() @ w.double().t()) if which == "x" else (x.double() @ v.double().t())
        third = ((rate.amax(1) - rate.amin(1)) ** 3 / 2).sum()
        s = 2.0 ** -6
        up = vocab.xent_forward(x + s * v, w, labels)[0] if which == "x" else vocab.xent_forward(x, w + s * v, labels)[0]
        down = vocab.xent_forward(x - s * v, w, labels)[0] if which == "x" else vocab.xent_forward(x, w - s * v, labels)[0]
        slope = (up.double() - down.double()).sum() / (2 * s)
        moved = 2 * U * ((x.abs().double() @ w.abs().double().t()).amax()) * 6 / s        # x + s v itself is rounded
        tol = s * s / 6 * third + 2 * e.loss_err.sum() * 2 / (2 * s) + moved
        assert abs(float(slope) - float((grad.double() * v.double()).sum())) <= float(tol), which


# ---- embedding rows -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,V,D", [((1,), 1, 1), ((3, 5), 7, 3), ((1,), 100, 4096), ((130,), 50, 65), ((4097,), 81, 128), ((2, 700), 3000, 264), ((70000,), 33, 8),
                                       ((9000,), 100000, 16), ((2000,), 300, 1003), ((64,), 5000, 1000), ((65,), 5000, 1000), ((7, 9), 3001, 65), ((40,), 2 ** 21, 3), ((5000,), 2 ** 20 - 2, 8), ((5000,), 2 ** 20 - 1, 8), ((300, 300), 2 ** 21, 2)])
def test_embed(shape, V, D, dtype):
    from gossipnet_amd import vocab
    t = TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(V + D)
    table = torch.randn(V, D, device=DEV, generator=g).to(t)
    ids = (torch.rand(shape, device=DEV, generator=g) ** 3 * (V + 1)).long()      # the first ids are much more frequent
    ids[torch.rand(shape, device=DEV, generator=g) < 0.1] = -1                    # (V itself is outside as well)
    s = torch.rand(shape, device=DEV, generator=g)
    dy = torch.randn(shape + (D,), device=DEV, generator=g).to(t)
    ok = (ids >= 0) & (ids < V)
    for use, i in ((s, ids), (None, ids.int())):
        y = vocab.embed_forward(i, table, 1.7, use)
        f = torch.where(ok, (use.double() if use is not None else 1.0) * 1.7, 0.0)[..., None]
        exact = torch.where(ok[..., None], table.double()[ids.clamp(0, V - 1)] * f, 0.0)
        tiny = 2.0 ** -25 if t == torch.float16 else 0.0
        near(y, exact, exact.abs() * (half_step(t) + 4 * U) + tiny, "y")
        keep = torch.randn(V, D, device=DEV, generator=g).to(t)
        seen = torch.zeros(V, dtype=torch.bool, device=DEV)
        seen[ids[ok]] = True
        dt, ds = vocab.embed_backward(i, dy, table, 1.7, use, need_dscale=True)
        sums, mags = torch.zeros(V, D, dtype=torch.float64, device=DEV), torch.zeros(V, D, dtype=torch.float64, device=DEV)
        count = torch.zeros(V, dtype=torch.float64, device=DEV)
        term = (dy.double() * f)[ok]
        sums.index_add_(0, ids[ok], term); mags.index_add_(0, ids[ok], term.abs()); count.index_add_(0, ids[ok], torch.ones_like(ids[ok]).double())
        err = mags * (count[:, None] + 4) * U + tiny
        near(dt, sums, err + sums.abs() * half_step(t) * (1 + 2.0 ** -6), "dtable")
        assert not bool(dt[~seen].any())
        out = keep.clone()
        assert vocab.embed_backward(i, dy, table, 1.7, use, out=out)[0] is out
        total = sums + keep.double()
        near(out, total, err + total.abs() * (half_step(t) + U) * (1 + 2.0 ** -6), "out")
        assert torch.equal(out[~seen], keep[~seen])
        dot = torch.where(ok, (dy.double() * table.double()[ids.clamp(0, V - 1)]).sum(-1) * 1.7, 0.0)
        mag = (dy.double() * table.double()[ids.clamp(0, V - 1)]).abs().sum(-1) * 1.7
        near(ds, dot, mag * (D + 4) * U, "dscale")


@pytest.mark.parametrize("V", [40, 4000])
@pytest.mark.parametrize("M", [15, 16, 17, 32, 33, 63, 64, 65, 129, 2048, 2049, 4096, 4097, 65537, 70000])
def test_embed_gradient_of_one_row_and_of_runs_around_the_hot_limit(M, V):
    """All tokens the same id; and runs of 15, 16, 17 and more tokens at every place of the sorted order."""
    from gossipnet_amd import vocab
    D = 24
    g = torch.Generator(device=DEV).manual_seed(M)
    dy = torch.randint(-8, 9, (M, D), device=DEV, generator=g).float()       # sums of small whole numbers: exact
    table = torch.zeros(V, D, device=DEV)
    ids = torch.full((M,), 17, device=DEV)
    for _ in range(2):
        want = torch.zeros(V, D, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())
        assert torch.equal(vocab.embed_backward(ids, dy, table)[0].double(), want)
        sizes = [15, 16, 17, 1, 31, 32, 33, 2, 16, 16, 48, 64, 200, 3, 17]
        ids = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(sizes, device=DEV))
        ids = ids.repeat(M // ids.numel() + 1)[:M][torch.randperm(M, device=DEV, generator=g)]


@pytest.mark.parametrize("V", [50, 3000])
def test_embed_strides(V):
    from gossipnet_amd import vocab
    table = torch.randn(V, 64, device=DEV, dtype=torch.bfloat16)
    ids = torch.randint(0, V, (200,), device=DEV)
    dy = torch.randn(200, 64, device=DEV, dtype=torch.bfloat16)
    wide, dwide = torch.zeros(V, 77, device=DEV, dtype=torch.bfloat16), torch.zeros(200, 99, device=DEV, dtype=torch.bfloat16)
    wide[:, 5:69], dwide[:, 1:65] = table, dy
    assert torch.equal(vocab.embed_forward(ids, wide[:, 5:69], 2.0), vocab.embed_forward(ids, table, 2.0))
    assert torch.equal(vocab.embed_forward(ids, table.t().contiguous().t(), 2.0), vocab.embed_forward(ids, table, 2.0))
    for a, b in zip(vocab.embed_backward(ids, dwide[:, 1:65], wide[:, 5:69], need_dscale=True), vocab.embed_backward(ids, dy, table, need_dscale=True)):
        assert torch.equal(a, b)
    one = dy[:1].expand(200, 64)
    assert torch.equal(vocab.embed_backward(ids, one, table)[0], vocab.embed_backward(ids, one.contiguous(), table)[0])
    assert torch.equal(vocab.embed_forward(ids[::2], table), vocab.embed_forward(ids[::2].contiguous(), table))


# ---- sizes, streams, graphs, all together ----------------------------------------------------------------------------
@pytest.mark.parametrize("V,D", [(2 ** 20 + 5, 4096), (2 ** 20, 4099)])
def test_tables_beyond_32_bit_offsets(V, D):
    from gossipnet_amd import vocab
    # 8.6 GB: element offsets beyond 2^32
    g = torch.Generator(device=DEV).manual_seed(2)
    table = torch.empty(V, D, device=DEV, dtype=torch.bfloat16)
    for a in range(0, V, 2 ** 17):
        table[a:a + 2 ** 17] = torch.randn(min(2 ** 17, V - a), D, device=DEV, generator=g) * 0.03
    ids = torch.tensor([0, V - 1, V - 5, 5, V - 1], device=DEV)
    y = vocab.embed_forward(ids, table)
    assert torch.equal(y, table[ids])
    dt, _ = vocab.embed_backward(ids, y, table)
    assert torch.equal(dt[V - 1], (2 * y[1].float()).bfloat16()) and torch.equal(dt[V - 5], y[2]) and int(dt.any(1).sum()) == 4
    del dt
    x, labels = y * 8, ids
    e_lse = torch.logsumexp(torch.cat([x.double() @ table[a:a + 2 ** 17].double().t() for a in range(0, V, 2 ** 17)], 1), 1)
    e_hit = (x.double() * table[ids].double()).sum(1)
    loss, lse, hit = vocab.xent_forward(x, table, labels)
    tol = (D + 8) * U * float((x.double().abs().sum(1) * 0.2).max()) + 200 * U * 20
    near(lse, e_lse, torch.full_like(e_lse, tol), "lse")
    near(hit, e_hit, torch.full_like(e_hit, tol), "hit")
    dx, dw = vocab.xent_backward(x, table, labels, lse, hit, torch.ones(5, device=DEV))
    for v in (0, 7, V - 5, V - 1):
        z = x.double() @ table[v].double()
        dz = torch.exp(z - e_lse) - (labels == v).double()
        want = dz @ x.double()
        bound = (dz.abs() @ x.double().abs()) * (2 * half_step(torch.bfloat16) + 2 * tol + 16 * U) + want.abs() * half_step(torch.bfloat16)
        bound += (torch.exp(z - e_lse) * 3 * tol) @ x.double().abs()
        near(dw[v], want, bound, "dw[%d]" % v)
    del dw
    want = torch.zeros(5, D, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(want)
    for a in range(0, V, 2 ** 17):
        wd = table[a:a + 2 ** 17].double()
        p = torch.exp(x.double() @ wd.t() - e_lse[:, None])
        want += p @ wd
        mag += p @ wd.abs()
    want -= table[ids].double()
    mag += table[ids].double().abs()
    near(dx, want, mag * (half_step(torch.bfloat16) + V * U + 3 * tol) + want.abs() * half_step(torch.bfloat16), "dx")


def _step(x, w, ids, tid, tl, table):
    """Embedding rows into features, both losses on them, gradients back into the table: one tied training step."""
    from gossipnet_amd import vocab
    h = vocab.embed_forward(ids, table, 2.0)
    f = x + h
    loss, lse, hit = vocab.xent_forward(f, w, ids)
    loss2, lse2, hit2 = vocab.distill_forward(f, w, tid, tl, 1.5)
    n = torch.full((), 1.0 / ids.numel(), device=x.device)
    dx, dw = vocab.xent_backward(f, w, ids, lse, hit, n)
    dx2, dw2 = vocab.distill_backward(f, w, tid, tl, lse2, hit2, n, 1.5)
    total = dw + dw2
    vocab.embed_backward(ids, dx + dx2, table, 2.0, out=total)
    return loss, loss2, total


def test_tied_training_step_against_autograd():
    """The operators together as a model uses them: a table that is both ends' weights, fp32, against autograd in 64 bits on the CPU."""
    M, V, D, K = 50, 120, 64, 4
    x, w, ids, _, logits = make(M, V, D, "f32", 20, K)
    labels = ids[:, 0].clone()
    labels[::6] = -1
    loss, loss2, total = _step(x, w, labels, ids, logits, w)
    W = w.double().cpu().requires_grad_()
    lab, i, tl = labels.cpu(), ids.cpu(), logits.double().cpu()
    ok = lab >= 0
    f = x.double().cpu() + torch.where(ok[:, None], W[lab.clamp_min(0)] * 2.0, torch.zeros((), dtype=torch.float64))
    z = f @ W.t()
    a = torch.where(ok, torch.logsumexp(z, 1) - z.gather(1, lab.clamp_min(0)[:, None])[:, 0], torch.zeros((), dtype=torch.float64))
    q = torch.log_softmax(tl / 1.5, 1)
    b = (q.exp() * (q - torch.log_softmax(z / 1.5, 1).gather(1, i))).sum(1)
    ((a + b).sum() / M).backward()
    # fp32 all the way: every value on the way is a sum of at most V (or D) terms; a factor of 64 for the chain's four products
    scale = float(W.grad.abs().max())
    assert float((loss.double().cpu() - a.detach()).abs().max()) <= 64 * V * U and float((loss2.double().cpu() - b.detach()).abs().max()) <= 64 * V * U
    assert float((total.double().cpu() - W.grad).abs().max()) <= 64 * V * U * scale


@pytest.mark.parametrize("sizes", [[(40, 600, 128), (300, 2000, 64)], [(40, 100, 64), (300, 81, 128)], [(20, 300, 2048), (2100, 81, 64)], [(20, 700, 131), (9, 3000, 75)]])
def test_other_streams_and_captured_graphs(sizes):
    """Eager calls on a side stream, and a captured step replayed with new inputs, two graphs in turn, eager work between them."""
    steps = []
    for seed, (M, V, D) in enumerate(sizes):
        x, w, ids, _, logits = make(M, V, D, "bf16", seed, 4)
        steps.append([x, w, ids[:, 0].contiguous(), ids, logits, w])
    eager = [_step(*s) for s in steps]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [_step(*s) for s in steps]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(eager, other):
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*s)
        graphs.append(g); outs.append(out)
    for turn in range(4):
        for s in steps:
            s[0].copy_(torch.randn_like(s[0], dtype=torch.float32) * (turn + 1))
            s[2].copy_(s[2].roll(turn + 1))
        eager = [_step(*s) for s in steps]
        for k in (0, 1, 0) if turn % 2 else (1, 0):
            graphs[k].replay()
            torch.cuda.synchronize()
            for p, q in zip(outs[k], eager[k]):
                assert torch.equal(p, q), (turn, k)
