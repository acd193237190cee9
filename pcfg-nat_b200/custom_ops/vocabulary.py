"""The vocabulary table at both ends of a model, and the step behind its backward pass.

    token_logprobs(logits, tokens, top=0, entropy=False, ignore_index=None)  -> TokenLogprobs
    embed_tokens(weight, tokens, scale=1.0, padding_idx=None)                -> [..., H]
    embed_tokens_backward(grad_out, tokens, grad_weight, ...)                -> grad_weight, added to in place
    clip_grad_norm_(grads, max_norm, out=None, grad_scale=1.0)               -> norm (float32, on the device)

``token_logprobs`` stands beside ``dag_logsoftmax_gather_inplace``: one token per row instead of a sentence's target list,
the logits left as they are, any of float32, float16 and bfloat16, with what scoring an answer and an entropy term want to
know of the row.  ``embed_tokens`` takes what ``glance_select`` gives (the decoder input of the second pass) and is a
step of ``runtime.GlanceStep``; its gradient can be added onto the projection's ``d weight`` where the table is shared.
The arguments are checked, outputs allocated with torch, and the kernels run on the tensors' device and its current stream;
nothing is copied to the host.  There is no CPU path, and no forward-mode derivative: inputs with a tangent are refused.
All can be captured into a CUDA graph.  One that is captured before anything of this package ran on its device has no status word:
what such a graph does with bad tokens is the same, but ``read_status`` does not tell of it.
"""
import array
import itertools
import math
from collections import namedtuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import _cabi
from . import pcfg_loss as _ops

MAX_TOP = 32  # PCFGNAT_MAX_TOP
MAX_INDEX = 2_146_435_072  # PCFGNAT_MAX_INDEX
_FLOAT_END = 2.0 ** 128 - 2.0 ** 103  # from here on a number rounds to infinity in float32, which the kernels get
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # PCFGNAT_DTYPE_*

def _first_derivative(backward):
    """``once_differentiable``, whose guard is only set up where a graph of the backward pass is asked for."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


TokenLogprobs = namedtuple("TokenLogprobs", "logprob entropy top_logprob top_index")


def _numbers(t, name):
    """The PCFGNAT_DTYPE_* of a CUDA tensor of floating numbers."""
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} must be a tensor")
    if not t.is_cuda:
        _ops._require_cuda()
        raise RuntimeError(f"{name} must be a CUDA tensor")
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise RuntimeError(f"{name} must be float32, float16 or bfloat16 (got {t.dtype})")
    return dt


class _Stay:
    """What ``_on`` gives for the current device: switching to it costs more than a small kernel."""

    def __enter__(self):
        pass

    def __exit__(self, *_):
        pass


_STAY = _Stay()


def _on(dev):
    return _STAY if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)  # the handle alone: no object is made for it


def _token_tensor(tokens, dev, shape=None):
    if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64 or tokens.device != dev:
        raise RuntimeError(f"tokens must be an int64 tensor on {dev}")
    if shape is not None and tokens.shape != shape:
        raise RuntimeError(f"tokens must have shape {tuple(shape)}")
    return tokens.contiguous()


def _optional_index(i, name):
    """(whether there is one, its value) of an index argument that may be None."""
    if i is None:
        return 0, 0
    i = int(i)
    if not -(1 << 63) <= i < 1 << 63:
        raise RuntimeError(f"{name} must be a 64-bit integer")
    return 1, i


def _status_of(dev):
    """The device's status word; none while a graph is captured before there is one (it would belong to that graph)."""
    if dev.index not in _ops._status and torch.cuda.is_current_stream_capturing():
        return None
    return _ops._status_ptr(dev)


def _rows(t):
    """(rows of each group, stride between groups, stride between rows) of a tensor seen as rows of its last dimension."""
    shape, stride = t.shape[:-1], t.stride()
    if t.numel() == 0:
        return 1, 0, 0
    inner, stride_inner = 1, 0
    k = len(shape) - 1
    while k >= 0:  # the trailing dimensions that one stride describes
        if shape[k] != 1:
            if inner == 1:
                stride_inner = stride[k]
            elif stride[k] != inner * stride_inner:
                break
            inner *= shape[k]
        k -= 1
    outer, stride_outer = 1, 0
    while k >= 0:
        if shape[k] != 1:
            if outer == 1:
                stride_outer = stride[k]
            elif stride[k] != outer * stride_outer:
                return None
            outer *= shape[k]
        k -= 1
    return inner, stride_outer, stride_inner


def _logits_rows(logits):
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_INDEX:
        raise RuntimeError(f"logits must be [..., V] with V >= 1, at most {MAX_INDEX}")
    if logits.is_contiguous():
        return logits.numel() // logits.shape[-1] or 1, 0, logits.shape[-1]
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        raise RuntimeError("the vocabulary must be the dimension of stride 1 of logits")
    rows = _rows(logits)
    if rows is None:
        raise RuntimeError("the rows of logits must lie at no more than two strides: call contiguous() first")
    return rows


def _token_logprobs(logits, tokens, top, entropy, ignore, keep):
    """The forward call: (logprob, entropy or None, top_logprob or None, top_index or None, kept or None)."""
    dt, dev = _numbers(logits, "logits"), logits.device
    inner, stride_outer, stride_inner = _logits_rows(logits)
    shape = logits.shape[:-1]
    tokens = _token_tensor(tokens, dev, shape)
    n = tokens.numel()
    with _on(dev):
        logprob = tokens.new_empty(shape, dtype=torch.float32)
        ent = torch.empty_like(logprob) if entropy else None
        top_lp, top_ix = (logprob.new_empty(shape + (top,)), tokens.new_empty(shape + (top,))) if top else (None, None)
        kept = logprob.new_empty(shape + (2,)) if keep else None
        ptr = lambda t: t.data_ptr() if t is not None else None
        rc = _cabi.lib().pcfgnat_token_logprobs(logits.data_ptr(), dt, n, inner, stride_outer, stride_inner, logits.shape[-1],
                                                tokens.data_ptr(), *ignore, top, logprob.data_ptr(), ptr(ent), ptr(top_lp),
                                                ptr(top_ix), ptr(kept), _status_of(dev), _stream(dev))
    _cabi.check(rc, "pcfgnat_token_logprobs")
    return logprob, ent, top_lp, top_ix, kept


class TokenLogprobsFunc(Function):
    """``token_logprobs`` under autograd: the logits are kept as they are, and read again by the backward."""

    @staticmethod
    def forward(ctx, logits, tokens, top, entropy, ignore):
        logprob, ent, top_lp, top_ix, kept = _token_logprobs(logits, tokens, top, entropy, ignore, True)
        ctx.save_for_backward(logits, tokens.contiguous(), kept, ent, top_ix)
        ctx.top, ctx.ignore = top, ignore
        ctx.set_materialize_grads(False)
        if top_ix is not None:
            ctx.mark_non_differentiable(top_ix)
        return logprob, ent, top_lp, top_ix

    @staticmethod
    @_first_derivative
    def backward(ctx, g_logprob, g_entropy, g_top, _):
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        _ops._no_tangents((g_logprob, g_entropy, g_top))
        logits, tokens, kept, ent, top_ix = ctx.saved_tensors
        V, dev = logits.shape[-1], logits.device
        inner, stride_outer, stride_inner = _logits_rows(logits)
        n = tokens.numel()
        # rows as far apart as the logits' own where those are padded: both then start at the same place of a 16-byte vector
        pitch = stride_inner if V <= stride_inner < V + 64 else V
        cont = lambda g: None if g is None else g.contiguous()
        g_logprob, g_entropy, g_top = cont(g_logprob), cont(g_entropy), cont(g_top)
        ptr = lambda t: t.data_ptr() if t is not None else None
        with _on(dev):
            d = logits.new_empty(logits.shape[:-1] + (pitch,))
            rc = _cabi.lib().pcfgnat_token_logprobs_backward(
                logits.data_ptr(), _DTYPES[logits.dtype], n, inner, stride_outer, stride_inner, V, tokens.data_ptr(), *ctx.ignore,
                ctx.top if g_top is not None else 0, kept.data_ptr(), ptr(ent), ptr(top_ix), ptr(g_logprob), ptr(g_entropy),
                ptr(g_top), d.data_ptr(), pitch, _status_of(dev), _stream(dev))
        _cabi.check(rc, "pcfgnat_token_logprobs_backward")
        return d if pitch == V else d[..., :V], None, None, None, None


def token_logprobs(logits, tokens, top=0, entropy=False, ignore_index=None):
    """Log probabilities of given tokens: ``logprob`` [...] float32 = log_softmax(logits)[tokens] of ``logits`` [..., V]
    (float32, float16 or bfloat16; rows at any strides, the vocabulary at stride 1) and ``tokens`` [...] int64.

    ``entropy``: also the row's entropy in nats.  ``top`` (up to 32): also its best alternatives, ``top_logprob`` and
    ``top_index`` [..., top], falling, equal ones by rising index.  What is not asked for is None in the result, a
    ``TokenLogprobs``.  Differentiable with respect to the logits through logprob, entropy and top_logprob; the gradient is
    formed in float32 (probabilities below 2^-126 count as 0) and rounded once, and the logits must still hold what the forward saw.

    Rows whose token is ``ignore_index`` (padding) are not read: logprob, entropy and top_logprob 0, top_index -1, gradient 0.
    -inf masks an entry: it is no alternative, and where fewer than ``top`` are left the rest is (-inf, -1).  A row of nothing
    but -inf: logprob -inf, entropy 0, gradient 0; one with NaN or +inf: NaN.  A token outside the vocabulary: logprob NaN and
    ``PCFGNAT_STATUS_BAD_INDEX`` in ``read_status``."""
    top = int(top)
    if not 0 <= top <= MAX_TOP:
        raise RuntimeError(f"top must be between 0 and {MAX_TOP}, got {top}")
    ignore = _optional_index(ignore_index, "ignore_index")
    _ops._no_tangents((logits,))
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*TokenLogprobsFunc.apply(logits, tokens, top, bool(entropy), ignore))
    return TokenLogprobs(*_token_logprobs(logits, tokens, top, entropy, ignore, False)[:4])


def _table(weight, name):
    """(PCFGNAT_DTYPE_*, V, H, numbers between rows) of a table."""
    dt = _numbers(weight, name)
    shape = weight.shape
    if len(shape) != 2 or not 1 <= shape[0] <= MAX_INDEX or not 1 <= shape[1] <= 1 << 20:
        raise RuntimeError(f"{name} must be [V, H] with 1 <= V <= {MAX_INDEX} and 1 <= H <= 2^20")
    V, H = shape
    apart, beside = weight.stride()
    if H > 1 and beside != 1 or V > 1 and apart < H:
        raise RuntimeError(f"the rows of {name} must be contiguous and apart")
    return dt, V, H, max(apart, H)


def _padding(given, rows):
    """An ``_optional_index`` as the row of a table of that many: a negative one counts from the table's end."""
    there, i = given
    if there and not -rows <= i < rows:
        raise RuntimeError(f"padding_idx must be between {-rows} and {rows - 1}, got {i}")
    return there, i + rows if i < 0 else i


def _finite(x, name):
    x = float(x)
    if not -_FLOAT_END < x < _FLOAT_END:
        raise RuntimeError(f"{name} must be finite in float32, got {x}")
    return x


def _embed(weight, tokens, scale, padding):
    dt, V, H, apart = _table(weight, "weight")
    if not -V <= padding[1] < V:
        _padding(padding, V)  # nothing to do here, but refused where the gradient would be
    dev = weight.device
    tokens = _token_tensor(tokens, dev)
    with _on(dev):
        out = weight.new_empty(tokens.shape + (H,))
        rc = _cabi.lib().pcfgnat_embed(weight.data_ptr(), dt, apart, V, H, tokens.data_ptr(), tokens.numel(), scale, out.data_ptr(),
                                       _status_of(dev), _stream(dev))
    _cabi.check(rc, "pcfgnat_embed")
    return out


def _embed_backward(g, tokens, d_weight, table, scale, padding, accumulate):  # on the tensors' device; table: as _table tells
    dev = g.device
    dt, V, H, apart = table
    n = tokens.numel()
    stride = H
    if not g.is_contiguous():
        rows = _rows(g) if H == 1 or g.stride(-1) == 1 else None
        if rows is None or rows[0] != n and n > 1:  # not rows at one stride
            g = g.contiguous()
        else:
            stride = rows[2]
    lib = _cabi.lib()
    nbytes = lib.pcfgnat_embed_backward_workspace_bytes(n, V, H)  # none for few positions
    ws = tokens.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = lib.pcfgnat_embed_backward(g.data_ptr(), _DTYPES[g.dtype], stride, tokens.data_ptr(), n, V, H, scale, *padding, d_weight.data_ptr(),
                                    dt, apart, int(accumulate), ws.data_ptr() if nbytes else None, nbytes, _status_of(dev), _stream(dev))
    _cabi.check(rc, "pcfgnat_embed_backward")
    return d_weight


class EmbedTokensFunc(Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, padding):
        out = _embed(weight, tokens, scale, padding)  # checks them
        ctx.save_for_backward(tokens.contiguous())
        V, H = ctx.shape = weight.shape
        ctx.scale, ctx.padding, ctx.table = scale, _padding(padding, V), (_DTYPES[weight.dtype], V, H, H)  # the gradient's, which is contiguous
        return out

    @staticmethod
    @_first_derivative
    def backward(ctx, grad_out):
        _ops._no_tangents((grad_out,))
        (tokens,) = ctx.saved_tensors
        with _on(grad_out.device):
            d = grad_out.new_empty(ctx.shape)
            return _embed_backward(grad_out, tokens, d, ctx.table, ctx.scale, ctx.padding, False), None, None, None


def embed_tokens(weight, tokens, scale=1.0, padding_idx=None):
    """``scale`` * weight[tokens]: [..., H] in the type of ``weight`` [V, H] (float32, float16 or bfloat16; formed in float32,
    rounded once) for ``tokens`` [...] int64.  Differentiable with respect to the table: its gradient is dense, summed in
    float32 by sorted tokens, the same for the same input at the same alignment; ``padding_idx`` has none, as with torch's embedding (-1: the table's last row).  A token outside
    the table: a row of NaN and ``PCFGNAT_STATUS_BAD_INDEX`` in ``read_status``, no gradient."""
    scale = _finite(scale, "scale")
    padding = _optional_index(padding_idx, "padding_idx")
    _ops._no_tangents((weight,))
    if isinstance(weight, torch.Tensor) and weight.requires_grad and torch.is_grad_enabled():
        return EmbedTokensFunc.apply(weight, tokens, scale, padding)
    return _embed(weight, tokens, scale, padding)


def embed_tokens_backward(grad_out, tokens, grad_weight, scale=1.0, padding_idx=None, accumulate=True):
    """Adds the gradient of ``embed_tokens`` onto ``grad_weight`` [V, H] and returns it: for a table that the output projection
    shares, whose ``d weight`` (float32 from ``proj_backward_products``, float16 from ``runtime.LossStep(proj_backward=True)``) it
    completes without a second dense tensor.  Rows whose token does not occur are not touched; in the others a float32 number below 2^-126, of the table or
    the sum, counts as 0.  ``accumulate=False``: every row is
    overwritten.  ``grad_weight`` is float32 or of ``grad_out``'s type."""
    _ops._no_tangents((grad_out, grad_weight))
    _numbers(grad_out, "grad_out")
    table = _table(grad_weight, "grad_weight")
    scale = _finite(scale, "scale")
    padding = _padding(_optional_index(padding_idx, "padding_idx"), table[1])
    dev = grad_out.device
    if grad_weight.device != dev or grad_weight.dtype not in (torch.float32, grad_out.dtype):
        raise RuntimeError("grad_weight must be float32 or of grad_out's type, on its device")
    tokens = _token_tensor(tokens, dev)
    if grad_out.shape != tokens.shape + (grad_weight.shape[1],):
        raise RuntimeError("grad_out must be [..., H] for tokens [...] and grad_weight [V, H]")
    with _on(dev):
        _embed_backward(grad_out.detach(), tokens, grad_weight.detach(), table, scale, padding, accumulate)
    torch.autograd.graph.increment_version(grad_weight)  # written in place: autograd's checks see it
    return grad_weight


def _dense(t):
    """Whether the numbers of t fill a piece of memory without gaps, in whatever order."""
    if t.is_contiguous():
        return True
    order = sorted((d for d in range(t.dim()) if t.shape[d] != 1), key=t.stride, reverse=True)
    want = 1
    for d in reversed(order):
        if t.stride(d) != want:
            return False
        want *= t.shape[d]
    return True


def _check_layouts(grads, outs):
    """Refuses pairs of which the n-th number in memory is not the n-th number of both."""
    for g, o in zip(grads, outs):
        if not _dense(g):
            raise RuntimeError("a gradient must be dense: call contiguous() first")
        # equal strides alone do not make the output dense: its shape may be another
        if not (o.is_contiguous() and g.is_contiguous()) and (o.stride() != g.stride() or o.shape != g.shape):
            raise RuntimeError("an output must have its gradient's layout: both contiguous, or of one shape and the same strides")


def clip_grad_norm_(grads, max_norm, out=None, grad_scale=1.0):
    """Clips gradients by their global norm, as the trainer does between the backward pass and the optimizer.

    norm = abs(``grad_scale``) * sqrt(sum of all squares); every gradient is multiplied by grad_scale * min(1, max_norm / (norm +
    1e-6)), in place, or into the tensors ``out`` of as many numbers each (of its gradient's type or float32: half-precision
    gradients into float32 master gradients, with ``grad_scale`` = 1 / loss scale; contiguous as their gradients, or of the same
    shape and strides).  ``grads``: a tensor or an iterable of
    tensors of one device, float32, float16 or bfloat16 mixed, any number of them, in any dense layout; None among them is skipped
    (with its output).  Returns the norm before clipping, a float32 tensor on the device; nothing is read back.

    ``max_norm=math.inf`` only measures and scales by ``grad_scale``, whatever the norm; 0 makes every gradient 0.  Squares are
    summed in float64 (those of half-precision numbers by eights in float32 first), in an order that does not depend on timing:
    sizes, types, alignment and the number of SMs decide it.  A norm of NaN makes every gradient NaN; an infinite one makes finite gradients 0."""
    _ops._require_cuda()
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise RuntimeError(f"max_norm must be 0 or more, got {max_norm}")
    if _FLOAT_END <= max_norm < math.inf:  # a limit all the same, where infinity is none
        max_norm = torch.finfo(torch.float32).max
    grad_scale = _finite(grad_scale, "grad_scale")
    listed = lambda g: [g] if isinstance(g, torch.Tensor) else list(g)
    grads = listed(grads)
    outs = grads if out is None else listed(out)
    if len(outs) != len(grads):
        raise RuntimeError("out must hold one tensor per gradient")
    _ops._no_tangents(itertools.chain(grads, outs))
    # one plain pass over the list for each question: a model has hundreds of gradients, and the kernels are done with them sooner
    every = grads if out is None else grads + outs
    try:
        at = list(map(torch.Tensor.data_ptr, every))
    except TypeError:
        there = [i for i, g in enumerate(grads) if g is not None]
        if len(there) == len(grads):  # not because of a gradient that is None
            raise RuntimeError("gradients and outputs must be tensors") from None
        grads = [grads[i] for i in there]
        return clip_grad_norm_(grads, max_norm, None if out is None else [outs[i] for i in there], grad_scale)
    n = len(grads)
    if n == 0:
        return torch.zeros((), dtype=torch.float32, device=torch.device("cuda", torch.cuda.current_device()))
    size = list(map(torch.Tensor.numel, every))
    index = set(map(torch.Tensor.get_device, every))
    if len(index) != 1 or min(index) < 0:
        raise RuntimeError("the gradients and outputs must be CUDA tensors on one device")
    kind = [t.dtype for t in every]
    types, out_types = set(kind[:n]), set(kind[-n:])
    if not _DTYPES.keys() >= types | out_types:
        raise RuntimeError("gradients and outputs must be float32, float16 or bfloat16")
    if not all(map(torch.Tensor.is_contiguous, every)):
        _check_layouts(grads, outs)
    host = lambda code, v: array.array(code, v)  # read before the call returns
    kinds = lambda k, of: host("i", [_DTYPES[k[0]]]) * n if len(of) == 1 else host("i", map(_DTYPES.__getitem__, k))
    src, src_kind, numel = host("Q", at[:n]), kinds(kind[:n], types), host("q", size[:n])
    dst, dst_kind = src, src_kind
    if out is not None:
        if size[:n] != size[n:]:
            raise RuntimeError("an output must have its gradient's shape")
        if out_types != {torch.float32} and any(k != j and k != torch.float32 for j, k in zip(kind[:n], kind[n:])):
            raise RuntimeError("an output must be of its gradient's type or float32")
        dst, dst_kind = host("Q", at[n:]), kinds(kind[n:], out_types)
    dev = grads[0].device
    lib = _cabi.lib()
    head = lambda a: a.buffer_info()[0]
    with _on(dev):
        nbytes = lib.pcfgnat_clip_grad_norm_workspace_bytes(n)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        rc = lib.pcfgnat_clip_grad_norm(n, head(src), head(src_kind), head(dst), head(dst_kind), head(numel), max_norm, grad_scale,
                                        ws.data_ptr(), nbytes, norm.data_ptr(), _stream(dev))
    if rc == _cabi.ERR_INVALID_ARGUMENT:
        raise RuntimeError("the outputs must not overlap one another or another gradient")
    _cabi.check(rc, "pcfgnat_clip_grad_norm")
    torch.autograd.graph.increment_version(outs)  # written in place: autograd's checks see it
    return norm
