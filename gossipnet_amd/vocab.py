"""The two ends of a model over a large vocabulary on the HIP library (csrc/embed.hip, csrc/vocab.hip): rows of a [V, D] table by
token id with the table's gradient, and softmax losses over the V rows of a [V, D] weight matrix with theirs.  Plain tensors in,
plain tensors out, forward and backward as two calls (as in fc.py); PyTorch only owns the memory.

    y = embed_forward(ids, table, scale)                          # features of the tokens
    loss, lse, hit = xent_forward(x, w, labels)                   # one fp32 loss per token; sum or average as needed
    dx, dw = xent_backward(x, w, labels, lse, hit, dloss, loss=loss)      # dloss: d(total) / d(loss), per token or one number
    embed_backward(ids, dy, table, scale, out=dw)                 # a table that is also w: its second gradient is added

Tokens may be laid out in any number of leading dimensions ([B, T] or flat); x, w, table, dy are float32, bfloat16 or float16,
all of a call of one type; ids and labels int32 or int64.  An id or label outside [0, V) means "no token here" (padding): it adds
nothing, whatever its row holds.  Every result is reproducible bit for bit.  The calls run on the current stream of the tensors' device and
may be captured into a graph; workspaces come from PyTorch's allocator for each call."""
import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # GNET_F32, GNET_BF16, GNET_F16


def _p(t):
    return t.data_ptr() if t is not None else None


# (torch.cuda.current_stream makes an object first: 2 us of a call that takes 8)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev):
    return _raw_stream(dev.index) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(dev, f, *args):
    """The library's f on the stream that is current on device dev (which is made the current one if it is not: torch.cuda.device costs
    microseconds that a small call feels)."""
    if _current() == dev.index:
        _lib.check(f(*args, _stream(dev)), f.__name__)
    else:
        with torch.cuda.device(dev):
            _lib.check(f(*args, _stream(dev)), f.__name__)


def _matrix(t, what, cols=None, dtype=None):
    """A [..., D] tensor as rows of D consecutive elements (a view where its layout allows it)."""
    shape = t.shape
    if len(shape) < 1 or t.dtype not in _TYPES:
        raise _lib.InvalidArgumentError("%s must be a float32, bfloat16 or float16 tensor with at least one dimension" % what)
    if cols is not None and shape[-1] != cols:
        raise _lib.InvalidArgumentError("%s must have %d columns, not %d" % (what, cols, shape[-1]))
    if dtype is not None and t.dtype != dtype:
        raise _lib.InvalidArgumentError("%s is %s where %s is expected" % (what, t.dtype, dtype))
    if shape[-1] == 0:
        raise _lib.InvalidArgumentError("%s has rows of no elements" % what)
    if len(shape) != 2:
        t = t.detach().reshape(-1, shape[-1])
    step, one = t.stride()
    if one != 1 or (step < t.shape[1] and t.shape[0] > 1):
        t = t.detach().contiguous()
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _on_device(first, *others):
    """The device of a call (after the checks of shapes and types).  others: tensors or None."""
    here = first.get_device()
    if here < 0:
        raise _lib.GnetError("the vocabulary operators have only device kernels: pass CUDA/HIP tensors")
    for t in others:
        if t is not None and t.get_device() != here:
            raise _lib.InvalidArgumentError("a tensor of shape %s is on %s where %s is expected" % (tuple(t.shape), t.device, first.device))
    return first.device


def _ids(t, what, shape=None):
    if t.dtype not in (torch.int32, torch.int64):
        raise _lib.InvalidArgumentError("%s must be int32 or int64, not %s" % (what, t.dtype))
    if shape is not None and t.shape != shape:
        raise _lib.InvalidArgumentError("%s has shape %s where %s is expected" % (what, tuple(t.shape), tuple(shape)))
    return t.contiguous()


def _overlap(a, b):
    """Whether two matrices of consecutive row elements share memory."""
    if not a.numel() or not b.numel():
        return False
    ends = [t.data_ptr() + ((t.shape[0] - 1) * _ld(t) + t.shape[1]) * t.element_size() for t in (a, b)]
    return a.data_ptr() < ends[1] and b.data_ptr() < ends[0]


def _per_token(t, what, shape):
    """fp32 values of the tokens' shape."""
    if t.shape != shape:
        raise _lib.InvalidArgumentError("%s has shape %s where %s is expected" % (what, tuple(t.shape), tuple(shape)))
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.detach().to(torch.float32).contiguous()


def _workspace(nbytes, device):
    """256-byte aligned scratch of this call.  From the caching allocator: ordered on the current stream, and part of the graph's own
    memory while one is captured, so that no two calls in flight share it."""
    if not nbytes:
        return None, None
    buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
    return buf, (buf.data_ptr() + 255) // 256 * 256


# ---- token rows ----------------------------------------------------------------------------------------------------
def embed_forward(ids, table, scale=1.0, token_scale=None):
    """y [*ids.shape, D] = scale * token_scale * table[ids]; zero rows where an id is outside [0, V).
    table [V, D]; token_scale: one factor per token, of ids' shape (a detection's score, for instance), or None."""
    if table.dim() != 2 or table.shape[0] < 1:
        raise _lib.InvalidArgumentError("table must be [V, D] with V >= 1")
    t = _matrix(table, "table")
    V, D = t.shape
    i = _ids(ids, "ids")
    s = _per_token(token_scale, "token_scale", ids.shape) if token_scale is not None else None
    dev = _on_device(t, i, s)
    y = t.new_empty(ids.shape + (D,))
    _call(dev, _lib.load().gnet_embed_forward, _p(i), int(i.dtype == torch.int64), _p(t), _ld(t), float(scale), _p(s), i.numel(), V, D,
          _TYPES[t.dtype], _p(y))
    return y


def embed_backward(ids, dy, table, scale=1.0, token_scale=None, need_dscale=False, out=None):
    """(dtable, dscale): gradients of embed_forward.  dtable [V, D] = scale * sum over the tokens of each id, in token order, of
    token_scale * dy.  out: a contiguous [V, D] gradient of table's type that dtable is added to and that is returned (added in fp32,
    rounded once; rows without a token keep their bits); not memory of dy, nor of table with need_dscale, which are read meanwhile.
    dscale (with need_dscale): fp32, of ids' shape, = scale * dy . table[ids]."""
    if table.dim() != 2 or table.shape[0] < 1:
        raise _lib.InvalidArgumentError("table must be [V, D] with V >= 1")
    t = _matrix(table, "table")
    V, D = t.shape
    i = _ids(ids, "ids")
    if dy.shape != ids.shape + (D,):
        raise _lib.InvalidArgumentError("dy has shape %s where %s is expected" % (tuple(dy.shape), tuple(ids.shape) + (D,)))
    g = _matrix(dy, "dy", D, t.dtype)
    s = _per_token(token_scale, "token_scale", ids.shape) if token_scale is not None else None
    if out is not None:
        if tuple(out.shape) != (V, D) or out.dtype != t.dtype or not out.is_contiguous():
            raise _lib.InvalidArgumentError("out must be a contiguous [%d, %d] tensor of type %s" % (V, D, t.dtype))
        if _overlap(out, g) or (need_dscale and _overlap(out, t)):
            raise _lib.InvalidArgumentError("out shares memory with %s, which is read while it is written" % ("dy" if _overlap(out, g) else "table"))
    dev = _on_device(t, i, g, s, out)
    dtable = out.detach() if out is not None else t.new_empty(V, D)
    M = i.numel()
    lib = _lib.load()
    dscale = torch.empty(ids.shape, dtype=torch.float32, device=dev) if need_dscale else None
    nbytes = lib.gnet_embed_workspace_bytes(M, D)
    buf, ws = _workspace(nbytes, dev)
    _call(dev, lib.gnet_embed_backward, _p(i), int(i.dtype == torch.int64), _p(g), _ld(g), float(scale), _p(s), M, V, D, _TYPES[t.dtype],
          _p(dtable), int(out is not None), _p(t), _ld(t), _p(dscale), ws, nbytes)
    return (out if out is not None else dtable), dscale


# ---- softmax losses over the vocabulary ------------------------------------------------------------------------------
def _features(x, w):
    if w.dim() != 2 or w.shape[0] < 1:
        raise _lib.InvalidArgumentError("w must be [V, D] with V >= 1")
    wm = _matrix(w, "w")
    return _matrix(x, "x", wm.shape[1], wm.dtype), wm


def _teacher(top_ids, top_logits, x, temperature):
    if not (temperature > 0 and temperature < float("inf")):
        raise _lib.InvalidArgumentError("temperature must be positive and finite, not %s" % (temperature,))
    lead = x.shape[:-1]
    if top_ids.dim() != len(lead) + 1 or top_ids.shape[:-1] != lead or top_ids.shape[-1] < 1:
        raise _lib.InvalidArgumentError("top_ids must be [*tokens, K] with K >= 1, tokens %s" % (tuple(lead),))
    return _ids(top_ids, "top_ids"), _per_token(top_logits, "top_logits", top_ids.shape)


def _loss_gradient(dloss, lead, device):
    """d(total) / d(loss) per token; one number (or a tensor without dimensions) stands for all of them."""
    if isinstance(dloss, (int, float)):
        return torch.full(lead, float(dloss), dtype=torch.float32, device=device)
    if dloss.dim() == 0:
        dloss = dloss.expand(lead)
    return _per_token(dloss, "dloss", lead)


def xent_forward(x, w, labels):
    """(loss, lse, hit), fp32, of labels' shape: softmax cross entropy of the logits x . w^T (x [*tokens, D], w [V, D]) against
    labels [*tokens], the logits' log-sum-exp and the label's logit.  All three are 0 where the label is outside [0, V)."""
    xm, wm = _features(x, w)
    lead = x.shape[:-1]
    i = _ids(labels, "labels", lead)
    dev = _on_device(wm, xm, i)
    (M, D), V = xm.shape, wm.shape[0]
    loss = torch.empty(lead, dtype=torch.float32, device=dev)
    lse, hit = torch.empty_like(loss), torch.empty_like(loss)
    lib = _lib.load()
    nbytes = lib.gnet_vocab_workspace_bytes(_p(wm), _ld(wm), M, V, D, 0, _TYPES[wm.dtype], 0)
    buf, ws = _workspace(nbytes, dev)
    _call(dev, lib.gnet_xent_forward, _p(xm), _ld(xm), _p(wm), _ld(wm), _p(i), int(i.dtype == torch.int64), M, V, D, _TYPES[wm.dtype],
          _p(loss), _p(lse), _p(hit), ws, nbytes)
    return loss, lse, hit


def xent_backward(x, w, labels, lse, hit, dloss, need_dx=True, need_dw=True, loss=None):
    """(dx, dw) of xent_forward, of x's and w's shapes and type, from its lse and hit (of the same x, w and labels: they are not looked
    at where a token's whole softmax is formed again) and the losses' gradient dloss (labels' shape, or a number or a tensor without
    dimensions for all tokens).  None for what is not needed.  loss: the forward's too; the gradient at a label is then dloss * expm1(-loss).  Without it, it
    comes from lse, whose fp32 rounding (2^-24 |lse|) is more than is left of 1 - softmax in a row whose loss is below that."""
    xm, wm = _features(x, w)
    lead = x.shape[:-1]
    i = _ids(labels, "labels", lead)
    known = _per_token(loss, "loss", lead) if loss is not None else None
    return _backward(xm, wm, i, None, 1.0, _per_token(lse, "lse", lead), _per_token(hit, "hit", lead), _loss_gradient(dloss, lead, x.device), x.shape, 0, need_dx, need_dw, known)


def distill_forward(x, w, top_ids, top_logits, temperature=1.0):
    """(loss, lse, hit), fp32: divergence of the student's softmax(x . w^T / temperature) from the teacher's softmax over its K best
    logits / temperature (top_ids, top_logits [*tokens, K]), the student's log-sum-exp [*tokens], and its logits / temperature at
    top_ids [*tokens, K].  Slots with an id outside [0, V) or a logit of -inf are left out; a token without slots has loss 0."""
    xm, wm = _features(x, w)
    lead = x.shape[:-1]
    i, t = _teacher(top_ids, top_logits, x, temperature)
    dev = _on_device(wm, xm, i, t)
    (M, D), V, K = xm.shape, wm.shape[0], i.shape[-1]
    loss = torch.empty(lead, dtype=torch.float32, device=dev)
    lse = torch.empty_like(loss)
    hit = torch.empty(lead + (K,), dtype=torch.float32, device=dev)
    lib = _lib.load()
    nbytes = lib.gnet_vocab_workspace_bytes(_p(wm), _ld(wm), M, V, D, K, _TYPES[wm.dtype], 0)
    buf, ws = _workspace(nbytes, dev)
    _call(dev, lib.gnet_distill_forward, _p(xm), _ld(xm), _p(wm), _ld(wm), _p(i), int(i.dtype == torch.int64), _p(t), float(temperature),
          M, V, D, K, _TYPES[wm.dtype], _p(loss), _p(lse), _p(hit), ws, nbytes)
    return loss, lse, hit


def distill_backward(x, w, top_ids, top_logits, lse, hit, dloss, temperature=1.0, need_dx=True, need_dw=True):
    """(dx, dw) of distill_forward, of x's and w's shapes and type (the teacher's logits get no gradient)."""
    xm, wm = _features(x, w)
    lead = x.shape[:-1]
    i, t = _teacher(top_ids, top_logits, x, temperature)
    return _backward(xm, wm, i, t, temperature, _per_token(lse, "lse", lead), _per_token(hit, "hit", i.shape), _loss_gradient(dloss, lead, x.device), x.shape, i.shape[-1], need_dx, need_dw)


def _backward(xm, wm, i, t, temperature, lse, hit, dloss, x_shape, K, need_dx, need_dw, loss=None):
    dev = _on_device(wm, xm, i, t, lse, hit, dloss, loss)
    (M, D), V, dt = xm.shape, wm.shape[0], _TYPES[wm.dtype]
    dx = xm.new_empty(x_shape) if need_dx else None
    dw = wm.new_empty(V, D) if need_dw else None
    if not (need_dx or need_dw):
        return dx, dw
    lib = _lib.load()
    nbytes = lib.gnet_vocab_workspace_bytes(_p(wm), _ld(wm), M, V, D, K, dt, 1)
    buf, ws = _workspace(nbytes, dev)
    ids64 = int(i.dtype == torch.int64)
    if t is None:
        _call(dev, lib.gnet_xent_backward_loss, _p(xm), _ld(xm), _p(wm), _ld(wm), _p(i), ids64, _p(loss), _p(lse), _p(hit), _p(dloss), M, V, D, dt,
              _p(dx), _p(dw), ws, nbytes)
    else:
        _call(dev, lib.gnet_distill_backward, _p(xm), _ld(xm), _p(wm), _ld(wm), _p(i), ids64, _p(t), float(temperature), _p(lse), _p(hit),
              _p(dloss), M, V, D, K, dt, _p(dx), _p(dw), ws, nbytes)
    return dx, dw
