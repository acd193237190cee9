"""token_logprobs, embed_tokens and its gradient, clip_grad_norm_: against their definitions in 64 bits, and their refusals.

Tolerances.  u = 2^-24 is half a step of float32, eps / 2 of the storage type one rounding to it.
* log p = (x - m) - log S: the difference and the subtraction round by u of their results, together below 3 u |log p|; log S inherits the relative error of
  S.  An exponential is off by 2^-22 (the hardware's) + 2 u |y| (y = (x - m) / log 2 rounded twice), which S averages with the
  weights p: at most 2^-22 + 2 u E|y|, E|y| <= 2 log2(V) <= 36 here; summing adds less than 256 u.  Together 2e-5.
* H = log S - U / S: the same relative error on U / S, at most 25 in nats: 2e-5 (1 + |U / S|), |U / S| <= H + log V.
* d x = p (-G - h (log p + H)) + g: 2e-5 of the sum of the absolute terms, and one rounding to the type.
* embedding: one product and one rounding.  Its gradient: a sum of n terms in float32 is off by at most n u sum|g|.
* clipping: the norm is rounded once from 64 bits; the factor and the product add 4 u.
"""
import ctypes
import importlib
import math

import pytest
import torch

from conftest import ROOT  # noqa: F401

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


@pytest.fixture(scope="session")
def voc(pkg):
    return importlib.import_module("pcfg_nat_b200.custom_ops.vocabulary")


@pytest.fixture(scope="session")
def lib(pkg):
    return importlib.import_module("pcfg_nat_b200._cabi").lib()


def _step(t):
    """Half a step of the type relative to the value, and half its smallest subnormal step."""
    f = torch.finfo(t)
    return f.eps / 2, f.tiny * f.eps / 2


def _close(got, want, slack, dtype=torch.float32):
    """|got - want| <= slack + one rounding to dtype, NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = odd & ~torch.isnan(want)
    assert torch.equal(got[same], want[same])
    rel, least = _step(dtype)
    slack = slack if isinstance(slack, torch.Tensor) else torch.full_like(want, slack)
    off = (got - want).abs() - (slack.double() + rel * (want.abs() + slack.double()) + least)
    off = off[~odd]
    assert off.numel() == 0 or off.max() <= 0, float(off.max())


def _logprobs64(logits, tokens, top=0, ignore=None):
    """The definition in 64 bits: (logprob, entropy, top_logprob, top_index, log p)."""
    x = logits.detach().double()
    V = x.shape[-1]
    odd = (torch.isnan(x) | (x == math.inf)).any(-1)
    empty = (x == -math.inf).all(-1)
    lp = torch.log_softmax(x.masked_fill((odd | empty)[..., None], 0.0), -1)
    lp = lp.masked_fill(empty[..., None], -math.inf).masked_fill(odd[..., None], math.nan)
    p = lp.exp()
    H = -torch.where(p == 0, 0.0, p * lp).sum(-1)
    inside = (tokens >= 0) & (tokens < V)
    got = lp.gather(-1, tokens.clamp(0, V - 1)[..., None])[..., 0].masked_fill(~inside, math.nan)
    value, index = torch.sort(lp.masked_fill(odd[..., None], -math.inf), dim=-1, descending=True, stable=True)
    value, index = value[..., :top], index[..., :top]
    index = torch.where(value == -math.inf, -1, index)
    short = top - value.shape[-1]
    if short > 0:
        value = torch.cat([value, value.new_full(value.shape[:-1] + (short,), -math.inf)], -1)
        index = torch.cat([index, index.new_full(index.shape[:-1] + (short,), -1)], -1)
    value = value.masked_fill(odd[..., None], math.nan)
    if ignore is not None:
        out = tokens == ignore
        got, H = got.masked_fill(out, 0.0), H.masked_fill(out, 0.0)
        value, index = value.masked_fill(out[..., None], 0.0), index.masked_fill(out[..., None], -1)
    return got, H, value, index, lp


def _check_forward(voc, logits, tokens, top, ignore=None):
    got = voc.token_logprobs(logits, tokens, top=top, entropy=True, ignore_index=ignore)
    lp, H, value, index, _ = _logprobs64(logits, tokens, top, ignore)
    room = lambda v: 2e-5 + 2 * U * v.nan_to_num(0, 0, 0).abs()
    _close(got.logprob, lp, room(lp))
    _close(got.entropy, H, 2e-5 * (1 + H.nan_to_num(0, 0, 0) + math.log(logits.shape[-1])))
    if top:
        assert torch.equal(got.top_index, index)
        _close(got.top_logprob, value, room(value))
    else:
        assert got.top_logprob is None and got.top_index is None
    return got


def _random_logits(shape, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)
    t = torch.randint(0, shape[-1], shape[:-1], generator=g, device="cuda")
    return x, t


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, V, top", [(1, 1, 1), (1, 2, 0), (3, 5, 8), (2, 7, 3), (5, 31, 32), (4, 33, 1), (300, 100, 4), (700, 1000, 5),
                                          (2, 2047, 32), (2, 2049, 7), (9, 4096, 20), (1, 39999, 5), (3, 40000, 32), (150, 40001, 2),
                                          (1, 128256, 20), (40, 151936, 8), (1200, 4100, 1)])
def test_logprobs_forward(voc, dtype, rows, V, top):
    x, t = _random_logits((rows, V), dtype, seed=rows + V)
    _check_forward(voc, x, t, top)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [8, 100, 1500, 40000])
def test_logprobs_of_equal_and_ordered_values(voc, dtype, V):
    """Ties everywhere, ties at the border only, rising and falling rows: the lowest index first."""
    ramp = torch.arange(V, device="cuda", dtype=torch.float32) / 512
    few = torch.arange(V, device="cuda") % 3
    last = torch.zeros(V, device="cuda")
    last[-5:] = 1
    signed = torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0)
    x = torch.stack([torch.zeros(V, device="cuda"), ramp, -ramp, few.float(), -few.float(), last, signed, ramp.floor()]).to(dtype)
    t = torch.arange(8, device="cuda") % V
    for top in (1, 5, 32):
        _check_forward(voc, x, t, top)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 6, 1000, 40003])
def test_logprobs_of_masked_rows(voc, dtype, V):
    """-inf, the type's lowest value, +inf and NaN: in one entry, in all but one, in all."""
    f = torch.finfo(dtype)
    x, _ = _random_logits((12, V), dtype, seed=V)
    t = torch.full((12,), V // 2, device="cuda")
    x[0] = -math.inf
    x[1] = f.min
    x[2] = -math.inf
    x[2, V // 2] = 1.5
    x[3] = f.min
    x[3, V // 3] = 0.25
    x[4, ::2] = -math.inf
    x[5, V - 1] = math.inf
    x[6, 0] = math.nan
    x[7, V // 2] = -math.inf
    x[8] = f.max
    x[9] = -math.inf
    x[9, V // 2] = f.min
    x[10] = -math.inf
    x[10, V // 3] = math.nan
    x[11, : V // 2] = f.min
    for top in (0, 3, 32):
        _check_forward(voc, x, t, top)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_of_far_apart_and_shifted_logits(voc, dtype):
    x, t = _random_logits((6, 5000), dtype, spread=1.0)
    x[0] += 1000
    x[1] -= 1000
    x[2, 17] = 300
    x[3] *= 5000
    x[4, :] = -30000
    x[4, 4321] = 30000
    _check_forward(voc, x, t, 6)


@gpu
def test_logprobs_masked_vocabulary_with_allowed_entries_close_together(voc):
    """More allowed entries than one list holds, all seen by a few threads; and fewer than asked for."""
    x = torch.full((3, 50000), -math.inf, device="cuda")
    x[0, 8:16] = torch.arange(8, device="cuda").float()
    for i, threads in ((1, 8), (2, 31)):
        x[i].view(-1, 4)[torch.arange(12500, device="cuda") % 256 < threads] = torch.randn(4, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    _check_forward(voc, x, t, 32)


@gpu
def test_logprobs_indices_ignored_rows_and_status(voc, ops):
    x, t = _random_logits((3, 4, 77), torch.float32)
    t[0, 0], t[1, 1], t[2, 2], t[2, 3] = -1, 77, 1 << 32, 5
    ops.read_status()
    _check_forward(voc, x, t, 3)
    assert ops.read_status() == 4
    t = torch.full((3, 4), 5, device="cuda")
    t[1] = -100
    x[1] = math.nan
    got = _check_forward(voc, x, t, 3, ignore=-100)
    assert torch.equal(got.logprob[1], torch.zeros(4, device="cuda")) and ops.read_status() == 0


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_of_strided_logits(voc, dtype):
    base, _ = _random_logits((4, 9, 1003), dtype)
    t = torch.randint(0, 990, (4, 9), device="cuda")
    for x in (base[..., :1001], base[..., 1:1000], base[:, 1:, 2:], base[::2], base[:, ::3, :990], base[:, 2], base[0, 0],
              base[:1].expand(4, 9, 1003), base.transpose(0, 1), base.view(2, 2, 9, 1003)):
        _check_forward(voc, x, t.new_zeros(x.shape[:-1]) + 3, 4)
    with pytest.raises(RuntimeError, match="stride 1"):
        voc.token_logprobs(base.transpose(1, 2), t.new_zeros((4, 1003)))
    with pytest.raises(RuntimeError, match="two strides"):
        voc.token_logprobs(base.view(2, 2, 9, 1003)[:, :1].expand(2, 3, 9, 1003)[:, :, ::2], t.new_zeros((2, 3, 5)))
    none = voc.token_logprobs(base[:0], t[:0], top=2, entropy=True)
    assert none.logprob.shape == (0, 9) and none.top_index.shape == (0, 9, 2)
    assert voc.token_logprobs(base[0, 0], t[0, 0]).logprob.shape == ()


@gpu
def test_logprobs_beyond_32_bit_offsets(voc):
    far = 3_000_000_000
    buf = torch.empty(far + 5000, dtype=torch.float16, device="cuda")
    x = buf.as_strided((2, 4999), (far, 1))
    x[0], x[1] = torch.randn(4999, device="cuda"), torch.randn(4999, device="cuda")
    t = torch.tensor([3, 4998], device="cuda")
    _check_forward(voc, x, t, 3)


def _grads64(logits, tokens, ignore, top, g_lp, g_h, g_top):
    lp0, H, _, index, lp = _logprobs64(logits, tokens, top, ignore)
    V = logits.shape[-1]
    p = lp.exp()
    add = torch.zeros_like(lp)
    total = torch.zeros_like(lp[..., :1])
    if g_lp is not None:
        inside = (tokens >= 0) & (tokens < V)
        add.scatter_add_(-1, tokens.clamp(0, V - 1)[..., None], torch.where(inside, g_lp, 0).double()[..., None])
        total += torch.where(inside, g_lp.double(), math.nan)[..., None]
    if g_top is not None:
        g = torch.where(index >= 0, g_top, 0).double()
        add.scatter_add_(-1, index.clamp(min=0), g)
        total += g.sum(-1, keepdim=True)
    h = g_h.double()[..., None] if g_h is not None else torch.zeros_like(total)
    lpf = torch.where(p == 0, 0.0, lp)
    d = p * (-total - h * (lpf + H[..., None])) + add
    size = p * (total.abs() + h.abs() * (lpf.abs() + H.abs()[..., None])) + add.abs()
    zero = (logits == -math.inf).all(-1)
    if ignore is not None:
        zero = zero | (tokens == ignore)
    return d.masked_fill(zero[..., None], 0.0), size.masked_fill(zero[..., None], 0.0)


def _check_backward(voc, logits, tokens, top=0, ignore=None, use="lht", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = logits.detach().requires_grad_(True)
    got = voc.token_logprobs(x, tokens, top=top, entropy="h" in use, ignore_index=ignore)
    draw = lambda t: torch.randn(t.shape, generator=g, device="cuda")
    outs, gs = [], dict(l=None, h=None, t=None)
    for key, t in (("l", got.logprob), ("h", got.entropy), ("t", got.top_logprob)):
        if key in use and t is not None:
            gs[key] = draw(t)
            outs.append((t, gs[key]))
    d, = torch.autograd.grad([o for o, _ in outs], [x], [v for _, v in outs])
    assert d.dtype == x.dtype
    want, size = _grads64(logits, tokens, ignore, top, gs["l"], gs["h"], gs["t"])
    # 2e-5 as above; x - m rounds by u |x - m|, at most 104 u where p is not below float32's least, and log S by as much again
    _close(d, want, (3.5e-5 * size).nan_to_num(0) + 1e-37, x.dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, V, top, use", [(1, 1, 1, "lht"), (2, 5, 3, "lht"), (3, 33, 0, "l"), (6, 1000, 32, "t"), (5, 1001, 4, "lht"),
                                               (4, 8192, 0, "h"), (3, 40000, 5, "lh"), (2, 39999, 2, "lht"), (200, 501, 1, "lt"),
                                               (2, 151936, 20, "lht")])
def test_logprobs_backward(voc, dtype, rows, V, top, use):
    x, t = _random_logits((rows, V), dtype, seed=rows * V)
    if rows > 1:
        t[0] = 1 % V
    _check_backward(voc, x, t, top, ignore=1 % V if rows > 1 else None, use=use)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_logprobs_backward_of_masked_and_strided_rows(voc, dtype):
    f = torch.finfo(dtype)
    x, t = _random_logits((2, 5, 1010), dtype)
    x[0, 0] = -math.inf
    x[0, 1, ::2] = -math.inf
    x[0, 2, 3:] = f.min
    x[0, 3] = -math.inf
    x[0, 3, 7] = 2.0
    t[0, 1], t[0, 3] = 4, 7
    t[1, 4] = 2000
    t.clamp_(max=999)
    for view in (x, x[..., :1001], x[:, :-1, 3:1003], x[:, ::2, :1000], x[..., 1:]):
        _check_backward(voc, view, t[:, : view.shape[1]], top=6)
    t[0, 4] = 1 << 33
    _check_backward(voc, x, t, top=2)
    bad = x[:, :, :1000].clone()
    bad[1, 1, 3], bad[1, 2, 4] = math.nan, math.inf
    _check_backward(voc, bad, t.clamp(max=999), top=2)
    _check_backward(voc, x[:1, :1].expand(2, 5, 1010), t.clamp(max=999), top=2)


@gpu
def test_logprobs_gradient_against_differences(voc):
    """d/dx of a weighted sum of all three outputs along random directions, differences of the definition in 64 bits."""
    x, t = _random_logits((4, 300), torch.float32, spread=1.5)
    g = torch.Generator(device="cuda").manual_seed(3)
    w = [torch.randn(s, generator=g, device="cuda") for s in ((4,), (4,), (4, 3))]
    leaf = x.clone().requires_grad_(True)
    got = voc.token_logprobs(leaf, t, top=3, entropy=True)
    ((got.logprob * w[0]).sum() + (got.entropy * w[1]).sum() + (got.top_logprob * w[2]).sum()).backward()
    value = lambda z: sum((a * b.double()).sum() for a, b in zip(_logprobs64(z, t, 3)[:3], w))
    for _ in range(4):
        v = torch.randn(x.shape, generator=g, device="cuda").double()
        step = 1e-5
        slope = (value(x.double() + step * v) - value(x.double() - step * v)) / (2 * step)
        # differences: step^2 of the third derivative, below 1e-7; the gradient 2e-5 of its terms
        assert abs(float((leaf.grad.double() * v).sum() - slope)) < 2e-5 * float((leaf.grad.double() * v).abs().sum()) + 1e-5


@gpu
def test_logprobs_refuse_a_changed_input_and_a_second_derivative(voc):
    x, t = _random_logits((2, 50), torch.float32)
    leaf = x.requires_grad_(True)
    y = leaf * 1.0
    out = voc.token_logprobs(y, t)
    y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprob.sum().backward()
    out = voc.token_logprobs(leaf, t)
    d, = torch.autograd.grad(out.logprob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@gpu
def test_logprobs_rows_of_a_pitched_gradient_keep_what_lies_behind(lib):
    x, t = _random_logits((3, 50), torch.float16)
    kept = torch.zeros((3, 2), device="cuda")
    lp, g = torch.empty(3, device="cuda"), torch.ones(3, device="cuda")
    d = torch.full((3, 56), 7.0, dtype=torch.float16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    assert lib.pcfgnat_token_logprobs(x.data_ptr(), 1, 3, 3, 0, 50, 50, t.data_ptr(), 0, 0, 0, lp.data_ptr(), None, None, None,
                                      kept.data_ptr(), None, st) == 0
    assert lib.pcfgnat_token_logprobs_backward(x.data_ptr(), 1, 3, 3, 0, 50, 50, t.data_ptr(), 0, 0, 0, kept.data_ptr(), None, None,
                                               g.data_ptr(), None, None, d.data_ptr(), 56, None, st) == 0
    assert torch.equal(d[:, 50:], torch.full((3, 6), 7.0, dtype=torch.float16, device="cuda")) and not (d[:, :50] == 7).any()


# ---- embedding


def _check_embed(voc, w, t, scale):
    got = voc.embed_tokens(w, t, scale=scale)
    V = w.shape[0]
    inside = (t >= 0) & (t < V)
    want = torch.where(inside[..., None], w.double()[t.clamp(0, V - 1)] * float(torch.tensor(scale, dtype=torch.float32)), math.nan)
    assert got.dtype == w.dtype
    _close(got, want, U * want.abs().nan_to_num(0, 0, 0), w.dtype)
    return got


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V, H, n", [(1, 1, 1), (5, 3, 4), (50, 8, 0), (1000, 512, 140), (40000, 512, 3000), (777, 301, 500), (33, 1024, 7),
                                     (100, 2050, 65), (9, 12, 40000)])
def test_embedding_forward(voc, dtype, V, H, n):
    w = torch.randn((V, H), device="cuda").to(dtype)
    t = torch.randint(0, V, (n,), device="cuda")
    _check_embed(voc, w, t, 1.0)
    _check_embed(voc, w, t.view(1, n), -math.sqrt(H))
    assert torch.equal(voc.embed_tokens(w, t), w[t])  # times 1 is exact


@gpu
def test_embedding_of_strided_tables_bad_tokens_and_odd_shapes(voc, ops):
    base = torch.randn((100, 72), device="cuda").half()
    base[3, 5], base[4, 6], base[5, 7] = math.nan, math.inf, -math.inf
    t = torch.arange(-2, 104, device="cuda").view(2, 53)
    ops.read_status()
    for w in (base[:, :64], base[:, 1:65], base[::2], base[1:, :71], base[:1]):
        _check_embed(voc, w, t, 3.0)
    assert ops.read_status() == 4
    assert voc.embed_tokens(base, torch.tensor(3, device="cuda")).shape == (72,)
    assert voc.embed_tokens(base, t[:, ::2][:, :3].clamp(0, 9).t()).shape == (3, 2, 72)
    with pytest.raises(RuntimeError, match="contiguous"):
        voc.embed_tokens(base.t(), t)


def _grad64(g, t, V, scale, padding):
    t, g = t.reshape(-1), g.reshape(-1, g.shape[-1]).double()
    keep = (t >= 0) & (t < V)
    if padding is not None:
        keep &= t != padding
    scale = float(torch.tensor(scale, dtype=torch.float32))
    d = torch.zeros((V, g.shape[1]), dtype=torch.float64, device=g.device).index_add_(0, t[keep], g[keep] * scale)
    size = torch.zeros_like(d).index_add_(0, t[keep], (g[keep] * scale).abs())
    count = torch.bincount(t[keep], minlength=V)[:, None].double()
    return d, (count + 3) * U * size


def _check_grad(voc, g, t, V, scale, padding, into=None):
    H = g.shape[-1]
    want, room = _grad64(g, t, V, scale, padding)
    d = torch.full((V, H), math.nan, dtype=into or g.dtype, device="cuda")
    voc.embed_tokens_backward(g, t, d, scale=scale, padding_idx=padding, accumulate=False)
    _close(d, want, room, d.dtype)
    start = torch.randn((V, H), device="cuda").to(into or g.dtype)
    more = start.clone()
    voc.embed_tokens_backward(g, t, more, scale=scale, padding_idx=padding)
    _close(more, want + start.double(), room + U * (want.abs() + start.double().abs()), d.dtype)
    seen = torch.zeros(V, dtype=torch.bool, device="cuda")
    keep = (t >= 0) & (t < V) & (t != (padding if padding is not None else -1))
    seen[t[keep]] = True
    assert torch.equal(more[~seen], start[~seen])  # rows without a token are not touched
    return d


@gpu
@pytest.mark.parametrize("dtype, into", [(t, t) for t in TYPES] + [(t, torch.float32) for t in TYPES[1:]])
@pytest.mark.parametrize("V, H, n, hot", [(1, 1, 1, 0), (5, 3, 4, 0), (50, 8, 0, 0), (1000, 512, 140, 0.5), (40000, 512, 5000, 0.7),
                                          (777, 301, 3000, 0.9), (33, 1024, 257, 0), (100, 2050, 65, 0), (3, 20, 40000, 0.3), (2000, 64, 33000, 1.0),
                                          (60000, 6, 1000, 0), (200000, 16, 2000, 0.2)])
def test_embedding_gradient(voc, dtype, into, V, H, n, hot):
    gen = torch.Generator(device="cuda").manual_seed(V + n)
    g = torch.randn((n, H), generator=gen, device="cuda").to(dtype)
    t = torch.randint(0, V, (n,), generator=gen, device="cuda")
    t = torch.where(torch.rand(n, generator=gen, device="cuda") < hot, V // 2, t)
    _check_grad(voc, g, t, V, 1.0, None, into)
    d = _check_grad(voc, g, t, V, 0.37, 0, into)
    again = torch.empty_like(d)
    voc.embed_tokens_backward(g, t, again, scale=0.37, padding_idx=0, accumulate=False)
    assert torch.equal(d, again)


@gpu
def test_embedding_gradient_of_sorted_sets(voc, ops):
    """One token only, padding only, every token once in falling order, bad tokens among others, runs that end at a piece's end."""
    V, H = 500, 24
    ops.read_status()
    for t in ([7] * 999, [0] * 100, list(range(499, -1, -1)), [5, -1, 500, 5, 1 << 40, 0, 499] * 31, [3] * 16 + [4] * 16 + [5] * 32 + [6],
              [1] + [9] * 63 + [2], [498] * 17 + [499] * 47):
        t = torch.tensor(t, device="cuda")
        for at in (t, t.flip(0), t.repeat(16), t.repeat_interleave(16), t.repeat_interleave(9).flip(0)):  # few positions, and many
            _check_grad(voc, torch.randn((len(at), H), device="cuda"), at, V, 2.0, 0)
    assert ops.read_status() == 4


@gpu
@pytest.mark.parametrize("n", [255, 256, 257, 1023, 1024, 1025, 2049, 8191, 33000])
def test_embedding_gradient_around_the_kernels_limits(voc, n):
    """One position more or less than a launch, a tile or a piece holds; a table beyond one window of a bucket's tokens."""
    for V, H in ((7, 5), (1025, 33), (140_001, 8)):
        t = torch.randint(0, V, (n,), device="cuda")
        t[: n // 3] = V - 1
        _check_grad(voc, torch.randn((n, H), device="cuda").half(), t, V, 1.5, 0, torch.float32)


@gpu
@pytest.mark.parametrize("n", [257, 5000, 600_000, 1_200_000])
@pytest.mark.parametrize("V", [1, 130, 150_000])
@pytest.mark.parametrize("which", ["evenly", "first", "only there", "nowhere else", "padding", "bad"])
def test_embedding_gradient_of_a_frequent_token(voc, ops, n, V, which):
    """Positions at even distances hold one token (so do all, a first part of them, no others, or only others do), or one that is left out."""
    ops.read_status()
    t = torch.randint(0, V, (n,), device="cuda")
    there = torch.arange(32, device="cuda") * n // 32
    token = {"padding": 0, "bad": V + 3}.get(which, V - 1)
    if which == "first":
        t[: n // 3] = token
    elif which == "only there":
        t[there] = token
    elif which == "nowhere else":
        other = t[there]
        t[:] = token
        t[there] = other
    else:
        t[torch.rand(n, device="cuda") < 0.6] = token
        t[there] = token
    _check_grad(voc, torch.randn((n, 4), device="cuda"), t, V, 1.0, 0 if which == "padding" else None)
    assert ops.read_status() == (4 if which == "bad" else 0)


@gpu
def test_embedding_gradient_through_autograd_and_of_broadcast_gradients(voc):
    w = torch.randn((300, 48), device="cuda").half().requires_grad_(True)
    t = torch.randint(0, 300, (4, 50), device="cuda")
    t[0] = 1
    voc.embed_tokens(w, t, scale=4.0, padding_idx=1).sum().backward()  # the gradient of a sum is one number, expanded
    want, room = _grad64(torch.ones((4, 50, 48), device="cuda"), t, 300, 4.0, 1)
    _close(w.grad, want, room, torch.float16)
    row = torch.randn(48, device="cuda").half()
    d, = torch.autograd.grad(voc.embed_tokens(w, t), w, row.expand(4, 50, 48))
    want, room = _grad64(row.expand(4, 50, 48), t, 300, 1.0, None)
    _close(d, want, room, torch.float16)
    base = torch.randn((4, 50, 60), device="cuda").half()
    for g in (base[..., :48], base[..., 3:51], torch.randn((50, 4, 48), device="cuda").half().transpose(0, 1),
              torch.randn((4, 48, 50), device="cuda").half().transpose(1, 2), base[:, :1, :48].expand(4, 50, 48)):
        want, room = _grad64(g, t, 300, 1.0, None)
        d, = torch.autograd.grad(voc.embed_tokens(w, t), w, g)
        _close(d, want, room, torch.float16)
    wide = torch.zeros((300, 64), device="cuda")
    voc.embed_tokens_backward(base[..., :48], t, wide[:, 8:56])
    want, room = _grad64(base[..., :48], t, 300, 1.0, None)
    _close(wide[:, 8:56], want, room)
    assert not wide[:, :8].any() and not wide[:, 56:].any()
    version = wide._version
    voc.embed_tokens_backward(base[..., :48], t, wide[:, 8:56])
    assert wide._version > version


@gpu
@pytest.mark.parametrize("n", [100, 3000])
def test_embedding_gradient_of_padding_is_not_read(voc, n):
    t = torch.randint(0, 50, (n,), device="cuda")
    t[::3], t[1::7] = 4, -5
    g = torch.randn((n, 24), device="cuda")
    g[(t == 4) | (t < 0)] = math.nan
    want, room = _grad64(torch.where(torch.isnan(g), 0, g), t, 50, 1.0, 4)
    d = voc.embed_tokens_backward(g, t, torch.empty((50, 24), device="cuda"), padding_idx=4, accumulate=False)
    _close(d, want, room)


@gpu
def test_embedding_gradient_against_differences(voc):
    w = torch.randn((20, 7), device="cuda", requires_grad=True)
    t = torch.randint(0, 20, (33,), device="cuda")
    c = torch.randn((33, 7), device="cuda")
    (voc.embed_tokens(w, t, scale=1.5) * c).sum().backward()
    v = torch.randn((20, 7), device="cuda")
    slope = ((w.detach().double() + v.double())[t] * 1.5 * c.double()).sum() - (w.detach().double()[t] * 1.5 * c.double()).sum()  # linear
    assert abs(float((w.grad.double() * v.double()).sum() - slope)) < 40 * U * float((w.grad.double() * v.double()).abs().sum()) + 1e-5


@gpu
def test_embedding_beyond_32_bit_offsets(voc):
    V, H = 4_300_000, 512
    w = torch.empty((V, H), dtype=torch.float16, device="cuda")
    t = torch.tensor([V - 1, 0, V - 1, 4_200_001], device="cuda")
    w[t] = torch.randn((4, H), device="cuda").half()
    assert torch.equal(voc.embed_tokens(w, t), w[t])
    g = torch.randn((4, H), device="cuda").half()
    w.fill_(math.nan)
    voc.embed_tokens_backward(g, t, w, accumulate=False)
    _close(w[V - 1], (g[0].double() + g[2].double()), 4 * U * (g[0].abs() + g[2].abs()).double(), torch.float16)
    assert torch.equal(w[0], g[1]) and torch.equal(w[4_200_001], g[3])
    assert int((w != 0).any(1).sum()) == 3


# ---- clipping


def _check_clip(voc, grads, max_norm, scale=1.0, out=None):
    before = [g.detach().clone() for g in grads]
    norm = voc.clip_grad_norm_(grads, max_norm, out=out, grad_scale=scale)
    s = float(torch.tensor(scale, dtype=torch.float32))
    want = abs(s) * math.sqrt(sum(float(b.double().square().sum()) for b in before))
    assert norm.dtype == torch.float32 and norm.shape == () and norm.is_cuda
    assert abs(float(norm) - want) <= 4 * U * want + 1e-45
    c = min(1.0, max_norm / (want + 1e-6)) * s
    for b, o, g in zip(before, grads if out is None else out, grads):
        _close(o, b.double() * c, 6 * U * (b.double() * c).abs(), o.dtype)
        if out is not None:
            assert torch.equal(g, b)


SIZES = [(1,), (7,), (8,), (0,), (), (3, 5), (1000,), (8192,), (8193,), (64, 513), (100001,)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_norm, scale", [(0.5, 1.0), (1e9, 1.0), (math.inf, 1.0), (1.0, 1 / 128), (0.0, 1.0), (2.0, -3.0)])
def test_clipping(voc, dtype, max_norm, scale):
    make = lambda: [torch.randn(s, device="cuda").to(dtype) for s in SIZES]
    _check_clip(voc, make(), max_norm, scale)
    grads = make()
    _check_clip(voc, grads, max_norm, scale, out=[torch.empty(g.shape, device="cuda") for g in grads])
    _check_clip(voc, grads, max_norm, scale, out=[torch.empty_like(g) for g in grads])
    flat = torch.randn(sum(math.prod(s) for s in SIZES) + 3, device="cuda").to(dtype)
    parts = [p.view(s) for p, s in zip(flat[3:].split([math.prod(s) for s in SIZES]), SIZES)]
    master = torch.empty(flat.numel() - 3, device="cuda")
    _check_clip(voc, parts, max_norm, scale, out=[p.view(s) for p, s in zip(master.split([math.prod(s) for s in SIZES]), SIZES)])
    _check_clip(voc, parts, max_norm, scale)


@gpu
def test_clipping_mixed_types_many_tensors_layouts_and_none(voc):
    grads = [torch.randn((i % 37 + 1,), device="cuda").to(TYPES[i % 3]) for i in range(2500)]
    _check_clip(voc, grads, 1.0)
    _check_clip(voc, [torch.randn((30, 50), device="cuda").t(), torch.randn((2, 8, 4, 4), device="cuda").to(memory_format=torch.channels_last)], 1.0)
    one = torch.randn(50, device="cuda")
    want = float(one.double().norm())
    assert abs(float(voc.clip_grad_norm_(one, math.inf)) - want) < 4 * U * want
    assert float(voc.clip_grad_norm_([], 1.0)) == 0 and float(voc.clip_grad_norm_([None, torch.zeros(0, device="cuda")], 1.0)) == 0
    _check_clip(voc, [g for g in [one, torch.zeros(9, device="cuda")]], 0.1)
    out = [torch.empty(50, device="cuda"), None]
    voc.clip_grad_norm_([one, None], 1.0, out=out)
    assert out[0].norm() <= 1.0 + 1e-5
    many = voc.clip_grad_norm_((g for g in grads), 1.0)
    assert abs(float(many) - 1.0) < 2.0 ** -7  # clipped to 1 before, rounded to bfloat16 at the worst


@gpu
def test_clipping_of_extreme_and_non_finite_gradients(voc):
    for dtype in (torch.float32, torch.bfloat16):  # squares beyond float32 in either direction
        _check_clip(voc, [torch.full((1000,), 1e25, device="cuda").to(dtype), torch.ones(3, device="cuda")], 1.0)
        tiny = torch.full((1000,), 1e-25, device="cuda").to(dtype)
        norm = voc.clip_grad_norm_([tiny], 1.0)
        want = float(tiny.double().norm())
        assert abs(float(norm) - want) <= 4 * U * want
    for bad in (math.nan, math.inf):
        g = [torch.ones(10, device="cuda"), torch.tensor([1.0, bad], device="cuda")]
        norm = voc.clip_grad_norm_(g, math.inf)  # measured only
        assert not math.isfinite(float(norm)) and torch.equal(g[0], torch.ones(10, device="cuda")) and g[1][0] == 1
        norm = voc.clip_grad_norm_(g, 1.0)
        assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
        if math.isnan(bad):
            assert all(bool(t.isnan().all()) for t in g)
        else:
            assert not g[0].any() and g[1][0] == 0 and g[1][1].isnan()


@gpu
def test_clipping_beyond_32_bit_offsets(voc):
    g = torch.zeros(2_200_000_000, dtype=torch.float16, device="cuda")
    g[0], g[-1], g[2_147_483_648] = 3, 4, 12
    norm = voc.clip_grad_norm_([g, torch.zeros(1, device="cuda")], 6.5)
    assert float(norm) == 13 and float(g[-1]) == 2 and float(g[0]) == 1.5 and float(g[2_147_483_648]) == 6
    assert int(torch.count_nonzero(g.view(-1, 100_000_000).float().abs().sum(1))) <= 3


# ---- together, on other streams, in graphs


def _tied_step(voc, table, hidden_weight, tokens, targets):
    """A training step of a toy model with a shared table: embed, one layer, logits, likelihood with an entropy term."""
    x = voc.embed_tokens(table, tokens, scale=math.sqrt(table.shape[1]), padding_idx=1)
    logits = torch.tanh(x @ hidden_weight) @ table.t()
    got = voc.token_logprobs(logits, targets, top=3, entropy=True, ignore_index=1)
    return -(got.logprob.sum() + 0.1 * got.entropy.sum() + 0.01 * got.top_logprob[..., 0].sum())


def _tied_step_plain(table, hidden_weight, tokens, targets):
    keep = (tokens != 1)[..., None]
    e = torch.where(keep, table[tokens], table[tokens].detach()) * math.sqrt(table.shape[1])
    lp = torch.log_softmax(torch.tanh(e @ hidden_weight) @ table.t(), -1)
    on = (targets != 1).to(lp.dtype)
    return -((lp.gather(-1, targets[..., None])[..., 0] - 0.1 * (lp.exp() * lp).sum(-1) + 0.01 * lp.max(-1).values) * on).sum()


@gpu
def test_a_training_step_of_all_operators(voc):
    g = torch.Generator(device="cuda").manual_seed(1)
    table = (torch.randn((211, 40), generator=g, device="cuda") / 6).requires_grad_(True)
    hw = (torch.randn((40, 40), generator=g, device="cuda") / 6).requires_grad_(True)
    tokens = torch.randint(0, 211, (3, 17), generator=g, device="cuda")
    targets = torch.randint(0, 211, (3, 17), generator=g, device="cuda")
    tokens[0, 9:], targets[0, 9:] = 1, 1
    loss = _tied_step(voc, table, hw, tokens, targets)
    loss.backward()
    norm = voc.clip_grad_norm_([table.grad, hw.grad], 0.7)
    t64, h64 = table.detach().double().requires_grad_(True), hw.detach().double().requires_grad_(True)
    want = _tied_step_plain(t64, h64, tokens, targets)
    want.backward()
    n64 = torch.cat([t64.grad.flatten(), h64.grad.flatten()]).norm()
    # float32 products of 40 and 211 terms around the operators, no cancellation: 1e-4 of the norm is far above their rounding
    assert abs(float(loss.detach() - want.detach())) < 1e-4 * abs(float(want.detach())) and abs(float(norm - n64)) < 1e-4 * float(n64)
    for got, w in ((table.grad, t64.grad), (hw.grad, h64.grad)):
        w = w * min(1.0, 0.7 / float(n64 + 1e-6))
        assert float((got - w).norm()) < 1e-4 * float(w.norm())


@gpu
def test_the_shared_tables_gradient_from_both_ends(voc, ops):
    """The projection's d weight from its own kernels, completed in place by the embedding's."""
    V, H = 200, 64
    w = (torch.randn((V, H), device="cuda") / 8).half()
    hidden = torch.randn((2, 12, H), device="cuda").half().requires_grad_(True)
    leaf = w.clone().requires_grad_(True)
    targets = torch.randint(0, V, (2, 5), device="cuda")
    match = ops.proj_logsoftmax_gather_with_grad(hidden, leaf, targets)
    match.sum().backward()
    d_weight = leaf.grad.float()
    tokens = torch.randint(0, V, (2, 12), device="cuda")
    g = torch.randn((2, 12, H), device="cuda").half()
    want, room = _grad64(g, tokens, V, 8.0, None)
    want = want + d_weight.double()
    got = voc.embed_tokens_backward(g, tokens, d_weight, scale=8.0)
    assert got is d_weight
    _close(got, want, room + U * want.abs())


@gpu
def test_the_glancing_step_embeds_the_second_passs_input(pkg, voc, ops, syn):
    """GlanceStep(embedding=...) against the operators one by one, over a new batch in the same graph, and the shared table's
    gradient from LossStep(proj_backward=True) completed by the embedding's."""
    runtime = importlib.import_module("pcfg_nat_b200.runtime")
    w = syn.Workload("ge", batch=4, vocab=2000, hidden=64, src_min=6, src_max=20, kind="glance")
    b = syn.make_batch(w, seed=5)
    weight = b.weight.cuda()
    prev = torch.where(torch.arange(b.L)[None, :] < b.output_length[:, None], 3, 1)
    batch = [b.hidden, b.links, b.output_length, b.targets, b.target_length, prev]
    gs = runtime.GlanceStep(weight, b.B, b.L, b.T, "cuda:0", embedding=weight, embed_scale=8.0)
    assert gs.kernels_per_step == runtime.GlanceStep.kernels_per_step + 1
    for tensors in (batch, [t.flip(0) for t in batch]):
        gs.load(*tensors)
        glance = gs.run()[3]
        tokens = glance["glat_prev_output_tokens"]
        assert torch.equal(glance["glat_embedded"], (weight[tokens].float() * 8).half())
        assert torch.equal(glance["glat_embedded"], voc.embed_tokens(weight, tokens, 8.0))
    plain = runtime.GlanceStep(weight, b.B, b.L, b.T, "cuda:0", use_graph=False)
    plain.load(*batch)
    assert "glat_embedded" not in plain.run()[3]
    with pytest.raises(RuntimeError, match="embedding must be"):
        runtime.GlanceStep(weight, b.B, b.L, b.T, "cuda:0", embedding=weight.cpu())
    ls = runtime.LossStep(weight, b.B, b.L, b.T, "cuda:0", proj_backward=True)
    ls.load(*batch[:5])
    d_weight = ls.run()[-1]
    start = d_weight.clone()
    g = torch.randn(tokens.shape + (64,), device="cuda").to(d_weight.dtype)
    voc.embed_tokens_backward(g, tokens, d_weight, scale=8.0, padding_idx=1)
    want, room = _grad64(g, tokens, 2000, 8.0, 1)
    want = want + start.double()
    _close(d_weight, want, room + U * want.abs(), d_weight.dtype)


@gpu
def test_on_another_stream_and_while_calls_overlap(voc):
    x, t = _random_logits((64, 20000), torch.bfloat16)
    w = torch.randn((20000, 128), device="cuda").bfloat16()
    g = torch.randn((64, 128), device="cuda").bfloat16()
    grads = [torch.randn((500, 500), device="cuda") for _ in range(3)]

    def calls():
        a = voc.token_logprobs(x, t, top=5, entropy=True)
        d = voc.embed_tokens_backward(g, t, torch.empty((20000, 128), device="cuda"), accumulate=False)
        out = [torch.empty_like(v) for v in grads]
        return [*a, voc.embed_tokens(w, t), d, voc.clip_grad_norm_(grads, 1.0, out=out), *out]

    want = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


@gpu
def test_captured_and_replayed(voc):
    """Two graphs over the same static inputs, replayed in turn and with new contents."""
    x, t = _random_logits((24, 5000), torch.float16)
    w = torch.randn((5000, 96), device="cuda").half()
    g = torch.randn((24, 96), device="cuda").half()
    gx, ge = torch.randn(24, device="cuda"), torch.randn(24, device="cuda")

    def calls():
        leaf, table = x.detach().requires_grad_(True), w.detach().requires_grad_(True)  # leaves of this call's own
        a = voc.token_logprobs(leaf, t, top=5, entropy=True, ignore_index=3)
        dx, = torch.autograd.grad([a.logprob, a.entropy], [leaf], [gx, ge])
        e = voc.embed_tokens(table, t, scale=2.0, padding_idx=3)
        dw, = torch.autograd.grad([e], [table], [g])
        out = [torch.empty(dx.shape, device="cuda"), torch.empty(dw.shape, device="cuda")]
        norm = voc.clip_grad_norm_([dx, dw], 1.0, out=out)
        return [v.detach() for v in (*a, dx, e, dw, norm, *out)]

    calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(calls())
        graphs.append(graph)
    for seed in range(3):
        fresh, ft = _random_logits((24, 5000), torch.float16, seed=seed)
        x.copy_(fresh)
        t.copy_(ft)
        t[seed] = 3
        for graph in graphs:
            graph.replay()
        want = calls()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- refusals (no GPU needed for the library's own)


def test_library_refuses_bad_arguments(lib):
    at = 16
    f = lambda rows=2, inner=2, V=5, top=0, logits=at, lp=at, tops=None: lib.pcfgnat_token_logprobs(
        logits, 0, rows, inner, 0, 5, V, at, 0, 0, top, lp, None, tops, tops, None, None, None)
    assert f(rows=-1) == f(inner=0) == f(V=0) == f(top=-1) == f(top=33, tops=at) == f(logits=None) == f(lp=None) == f(top=1) == -1
    assert f(rows=1 << 31) == -5 and f(rows=0) == 0
    b = lambda pitch=5, kept=at, g_h=None, g_top=None, top=0: lib.pcfgnat_token_logprobs_backward(
        at, 0, 2, 2, 0, 5, 5, at, 0, 0, top, kept, None, None, at, g_h, g_top, at, pitch, None, None)
    assert b(pitch=4) == b(kept=None) == b(g_h=at) == b(g_top=at, top=1) == -1
    assert lib.pcfgnat_embed(at, 0, 4, 0, 4, at, 1, 1.0, at, None, None) == -1
    assert lib.pcfgnat_embed(None, 0, 4, 4, 4, at, 1, 1.0, at, None, None) == -1
    assert lib.pcfgnat_embed(at, 3, 4, 4, 4, at, 1, 1.0, at, None, None) == -2
    need = lib.pcfgnat_embed_backward_workspace_bytes(1000, 4, 4)
    assert need > 0 and lib.pcfgnat_embed_backward_workspace_bytes(10, 4, 4) == 0
    e = lambda dtype=1, into=0, n=1000, ws=need, d=at, stride=4: lib.pcfgnat_embed_backward(
        at, dtype, 4, at, n, 4, 4, 1.0, 0, 0, d, into, stride, 0, at, ws, None, None)
    assert e(d=None) == e(stride=3) == e(n=-1) == -1 and e(into=2) == e(dtype=3) == -2 and e(ws=need - 1) == -4 and e(n=1 << 31) == -5


def test_library_refuses_overlapping_gradients(lib):
    def call(src, dst, size, sdt=0, ddt=0, norm=64, limit=1.0, room=1 << 20):
        n = len(src)
        arr = lambda t, v: (t * n)(*v)
        return lib.pcfgnat_clip_grad_norm(n, arr(ctypes.c_void_p, src), arr(ctypes.c_int, [sdt] * n), arr(ctypes.c_void_p, dst),
                                          arr(ctypes.c_int, [ddt] * n), arr(ctypes.c_int64, size), limit, 1.0, 64, room, norm, None)

    base = 1 << 20
    assert call([base, base], [base, base], [4, 4]) == -1                      # the same tensor twice
    assert call([base, base + 12], [base, base + 12], [4, 4]) == -1            # neighbours that share a number
    assert call([base], [base + 8], [4]) == -1                                 # an output over its own source, shifted
    assert call([base, base + 64], [base + 128, base], [4, 4]) == -1           # an output over another gradient
    assert call([base], [base], [-1]) == call([0], [0], [1]) == call([base], [base], [4], norm=None) == -1
    assert call([base], [base], [4], limit=-1.0) == call([base], [base], [4], limit=math.nan) == -1
    assert call([base], [base], [4], sdt=1, ddt=0) == call([base], [base + 64], [4], sdt=0, ddt=1) == call([base], [base], [4], 3, 3) == -2
    assert call([base], [base], [4], room=0) == -4


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_operators_refuse_to_run_without_cuda(voc):
    w, t = torch.zeros((4, 3)), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: voc.token_logprobs(w, t), lambda: voc.embed_tokens(w, t), lambda: voc.embed_tokens_backward(w, t, w),
                 lambda: voc.clip_grad_norm_([w], 1.0)):
        with pytest.raises(RuntimeError, match="You need GPU"):
            call()


def test_argument_checks_that_need_no_gpu(voc):
    w, t = torch.zeros((4, 3)), torch.zeros(4, dtype=torch.int64)
    for bad in (-1, 33):
        with pytest.raises(RuntimeError, match="top must be"):
            voc.token_logprobs(w, t, top=bad)
    for call in (lambda: voc.embed_tokens(w, t, scale=math.nan), lambda: voc.embed_tokens(w, t, scale=math.inf)):
        with pytest.raises(RuntimeError, match="scale must be finite"):
            call()
    with pytest.raises(RuntimeError, match="64-bit"):
        voc.embed_tokens(w, t, padding_idx=1 << 63)


def test_row_descriptions(voc):
    a = torch.zeros((4, 6, 10))
    assert voc._rows(a) == (24, 0, 10) and voc._rows(a[..., :7]) == (24, 0, 10)
    assert voc._rows(a[:, 1:]) == (5, 60, 10) and voc._rows(a[:, ::2]) == (12, 0, 20)
    assert voc._rows(a[::2, 1:, :3]) == (5, 120, 10) and voc._rows(a[:1]) == (6, 0, 10)
    assert voc._rows(a.transpose(0, 1)) == (4, 10, 60) and voc._rows(a[0, 0]) == (1, 0, 0)
    assert voc._rows(a[:1].expand(3, 6, 10)) == (6, 0, 10) and voc._rows(a[:0]) == (1, 0, 0)
    assert voc._rows(a.view(2, 2, 6, 10)[:, :1].expand(2, 3, 6, 10)[:, :, ::2]) is None
    assert voc._dense(a.transpose(0, 2)) and not voc._dense(a[:, 1:]) and not voc._dense(a[:1].expand(3, 6, 10)) and voc._dense(a[0, 0, 0])


@gpu
def test_refusals(voc):
    x, t = _random_logits((2, 8), torch.float32)
    cases = [
        (lambda: voc.token_logprobs(x.double(), t), "float32, float16 or bfloat16"),
        (lambda: voc.token_logprobs(x.cpu(), t), "CUDA tensor"),
        (lambda: voc.token_logprobs(x, t.int()), "int64"),
        (lambda: voc.token_logprobs(x, t.cpu()), "int64"),
        (lambda: voc.token_logprobs(x, t[:1]), "shape"),
        (lambda: voc.token_logprobs(x[:, :0], t), "V >= 1"),
        (lambda: voc.embed_tokens(x, t.float()), "int64"),
        (lambda: voc.embed_tokens(x[0], t), r"\[V, H\]"),
        (lambda: voc.embed_tokens(x[:, :0], t), r"\[V, H\]"),
        (lambda: voc.embed_tokens(x[:1].expand(4, 8), t), "apart"),
        (lambda: voc.embed_tokens_backward(x, t, torch.zeros((5, 7), device="cuda")), "grad_out must be"),
        (lambda: voc.embed_tokens_backward(x.half(), t, torch.zeros((5, 8), device="cuda").bfloat16()), "grad_weight must be"),
        (lambda: voc.clip_grad_norm_([x, x], 1.0), "overlap"),
        (lambda: voc.clip_grad_norm_([x], 1.0, out=[x[:1]]), "shape"),
        (lambda: voc.clip_grad_norm_([x], 1.0, out=[x.half()]), "type or float32"),
        (lambda: voc.clip_grad_norm_([x], 1.0, out=[]), "one tensor per gradient"),
        (lambda: voc.clip_grad_norm_([x], 1.0, out=[None]), "must be tensors"),
        (lambda: voc.clip_grad_norm_([x, 3.0], 1.0), "must be tensors"),
        (lambda: voc.clip_grad_norm_([x, t.float().cpu()], 1.0), "on one device"),
        (lambda: voc.clip_grad_norm_([x[:, ::2]], 1.0), "dense"),
        (lambda: voc.clip_grad_norm_([x[:1].expand(3, 8)], 1.0), "dense"),
        (lambda: voc.clip_grad_norm_([x], -1.0), "max_norm"),
        (lambda: voc.clip_grad_norm_([x], math.nan), "max_norm"),
        (lambda: voc.clip_grad_norm_([x.long()], 1.0), "float32, float16 or bfloat16"),
        (lambda: voc.clip_grad_norm_([x], 1.0, out=[torch.empty((8, 2), device="cuda").t()]), "layout"),
    ]
    for call, match in cases:
        with pytest.raises(RuntimeError, match=match):
            call()


def _pairs_of_equal_strides():
    """Gradients and outputs of equal strides and as many numbers, but of other shapes: the outputs have gaps."""
    make = lambda device: [
        (torch.zeros((4, 3, 2), device=device).permute(2, 1, 0), torch.full((6, 3, 2), 7.0, device=device)[:, :2].permute(2, 1, 0)),
        (torch.zeros((2, 3), device=device).t(), torch.full((3, 3), 7.0, device=device)[:, :2].t())]
    return make


def test_clipping_asks_for_outputs_of_one_layout(voc):
    for g, o in _pairs_of_equal_strides()("cpu"):
        assert g.stride() == o.stride() and g.numel() == o.numel() and voc._dense(g) and not voc._dense(o)
        with pytest.raises(RuntimeError, match="layout"):
            voc._check_layouts([g], [o])
        voc._check_layouts([g], [torch.empty_like(g)])
        voc._check_layouts([g], [g])
    flat, one = torch.zeros(12), torch.zeros(3, 4)
    voc._check_layouts([flat], [one])  # contiguous ones may be of another shape
    for g, o in ((one.t(), flat), (flat, one.t()), (one.t(), torch.zeros(4, 3))):
        with pytest.raises(RuntimeError, match="layout"):
            voc._check_layouts([g], [o])
    with pytest.raises(RuntimeError, match="dense"):
        voc._check_layouts([one[:, ::2]], [one[:, ::2]])


@gpu
def test_clipping_leaves_gaps_of_refused_outputs_alone(voc):
    for g, o in _pairs_of_equal_strides()("cuda"):
        with pytest.raises(RuntimeError, match="layout"):
            voc.clip_grad_norm_([g], 1.0, out=[o])
        assert bool((o._base == 7).all())
    g = torch.randn((2, 3), device="cuda").t()
    _check_clip(voc, [g], 0.5, out=[torch.empty_like(g)])


def test_library_refuses_tables_and_lists_whose_indices_could_leave_32_bits(lib, voc):
    limit, at, room = voc.MAX_INDEX, 16, 1 << 62
    e = lambda n=1, V=4: lib.pcfgnat_embed_backward(at, 1, 4, at, n, V, 4, 1.0, 0, 0, at, 0, 4, 0, at, room, None, None)
    for beyond in (limit + 1, (1 << 31) - 130, (1 << 31) - 1, 1 << 31):
        assert e(n=beyond) == e(V=beyond) == -5
    # at the limit: the last warp's share of the sorted list, and what a lane looks ahead
    share = -(-(-(-limit // (2048 * 8))) // 8) * 8
    begin = (limit - 1) // share * share
    assert begin + share + 64 < 1 << 31 and limit + 127 < 1 << 31


def test_tables_beyond_the_limit_are_refused_by_shape(voc, monkeypatch):
    monkeypatch.setattr(voc, "_numbers", lambda t, name: 1)  # a tensor without memory stands in for the table
    for V in (voc.MAX_INDEX + 1, (1 << 31) - 1):
        with pytest.raises(RuntimeError, match="must be"):
            voc._table(torch.empty((V, 2), device="meta"), "weight")
    assert voc._table(torch.empty((voc.MAX_INDEX, 2), device="meta"), "weight") == (1, voc.MAX_INDEX, 2, 2)


def test_rows_of_logits_whose_indices_could_leave_32_bits_are_refused(lib, voc):
    limit, at = voc.MAX_INDEX, 16
    for V in (limit + 1, (1 << 31) - 511, (1 << 31) - 1):  # the gradient's strided loop steps up to 512 beyond the row
        assert lib.pcfgnat_token_logprobs(at, 1, 1, 1, 0, V, V, at, 0, 0, 0, at, None, None, None, None, None, None) == -5
        assert lib.pcfgnat_token_logprobs_backward(at, 1, 1, 1, 0, V, V, at, 0, 0, 0, at, None, None, at, None, None, at, V, None, None) == -5
        with pytest.raises(RuntimeError, match="V >= 1, at most"):
            voc._logits_rows(torch.empty((1, V), device="meta"))
    assert voc._logits_rows(torch.empty((2, limit), device="meta")) == (2, 0, limit) and limit + 4 * 512 < 1 << 31


def test_padding_outside_the_table_is_refused(voc, monkeypatch):
    monkeypatch.setattr(voc, "_numbers", lambda t, name: 0)  # the table need not be on a GPU to be refused
    w, t = torch.zeros((4, 3)), torch.zeros(4, dtype=torch.int64)
    for bad in (4, -5, 1 << 40):
        with pytest.raises(RuntimeError, match="padding_idx must be between -4 and 3"):
            voc.embed_tokens(w, t, padding_idx=bad)
        with pytest.raises(RuntimeError, match="padding_idx must be between -4 and 3"):
            voc.embed_tokens(w.clone().requires_grad_(True), t, padding_idx=bad)
    given = lambda i: voc._padding(voc._optional_index(i, "padding_idx"), 4)
    assert given(None) == (0, 0) and given(-4) == (1, 0) and given(-1) == (1, 3) and given(3) == (1, 3) and given(0) == (1, 0)


@gpu
@pytest.mark.parametrize("n", [50, 700])
@pytest.mark.parametrize("padding", [None, 0, 5, -1, -6])
def test_padding_counts_from_the_end_as_torchs_does(voc, ops, n, padding):
    ops.read_status()
    w = torch.randn((6, 4), device="cuda", requires_grad=True)
    t = torch.randint(0, 6, (n,), device="cuda")
    g = torch.randn((n, 4), device="cuda")
    want, = torch.autograd.grad(torch.nn.functional.embedding(t, w.double(), padding_idx=padding), w, g.double())
    index = padding if padding is None or padding >= 0 else padding + 6
    _, room = _grad64(g, t, 6, 1.0, index)
    d, = torch.autograd.grad(voc.embed_tokens(w, t, padding_idx=padding), w, g)
    _close(d, want.double(), room + U * want.double().abs())  # torch's is rounded once as it leaves 64 bits
    direct = voc.embed_tokens_backward(g, t, torch.empty_like(w).detach(), padding_idx=padding, accumulate=False)
    assert torch.equal(direct, d) and ops.read_status() == 0
    for bad in (6, -7):
        with pytest.raises(RuntimeError, match="padding_idx must be between"):
            voc.embed_tokens_backward(g, t, torch.zeros((6, 4), device="cuda"), padding_idx=bad)


def test_factors_beyond_float32_are_refused(voc):
    w, t = torch.zeros((4, 3)), torch.zeros(4, dtype=torch.int64)
    for bad in (1e39, -1e39, 3.5e38):
        with pytest.raises(RuntimeError, match="scale must be finite"):
            voc.embed_tokens(w, t, scale=bad)
        with pytest.raises(RuntimeError, match="grad_scale must be finite"):
            voc._finite(bad, "grad_scale")
    last = math.nextafter(2.0 ** 128 - 2.0 ** 103, 0)
    assert math.isfinite(ctypes.c_float(last).value) and math.isinf(ctypes.c_float(2.0 ** 128 - 2.0 ** 103).value)
    assert voc._finite(last, "scale") == last and voc._finite(1, "scale") == 1.0 and voc._finite(1e-50, "scale") == 1e-50


@gpu
def test_factors_beyond_float32_are_refused_by_every_operator(voc):
    w, t = torch.ones((4, 3), device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (1e39, -math.inf, math.nan):
        for call in (lambda: voc.embed_tokens(w, t, scale=bad), lambda: voc.clip_grad_norm_(w, 1.0, grad_scale=bad),
                     lambda: voc.embed_tokens_backward(torch.ones((4, 3), device="cuda"), t, w, scale=bad)):
            with pytest.raises(RuntimeError, match="scale must be finite"):
                call()
    assert bool((w == 1).all())
    assert torch.equal(voc.embed_tokens(w, t, scale=3e38), w * 3e38)


@gpu
@pytest.mark.parametrize("limit", [3e38, 1e39, 1e300])
def test_a_finite_limit_beyond_float32_is_a_limit(voc, limit):
    """A norm of NaN makes every gradient NaN and an infinite one makes them 0 whatever the limit is, unless there is none."""
    g = torch.tensor([1.0, math.nan], device="cuda")
    assert math.isnan(float(voc.clip_grad_norm_(g, limit))) and bool(g.isnan().all())
    g = torch.tensor([1.0, math.inf], device="cuda")
    assert float(voc.clip_grad_norm_(g, limit)) == math.inf and g[0] == 0 and g[1].isnan()
    g = torch.tensor([3.0, 4.0], device="cuda")
    assert float(voc.clip_grad_norm_(g, limit)) == 5 and g.tolist() == [3.0, 4.0]


def test_forward_mode_tangents_are_refused(voc, monkeypatch):
    monkeypatch.setattr(voc._ops, "_require_cuda", lambda: None)
    w, t = torch.ones((4, 3)), torch.zeros(4, dtype=torch.int64)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: voc.token_logprobs(dual, t), lambda: voc.embed_tokens(dual, t), lambda: voc.embed_tokens_backward(dual, t, w),
                     lambda: voc.embed_tokens_backward(w, t, dual), lambda: voc.clip_grad_norm_(dual, 1.0),
                     lambda: voc.clip_grad_norm_([w, None], 1.0, out=[dual, None])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        voc._ops._no_tangents((w, t, None))  # others go on while a level is open
    voc._ops._no_tangents((dual,))


@gpu
def test_forward_mode_tangents_are_refused_before_anything_is_written(voc):
    w, t = torch.ones((4, 3), device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w.clone(), torch.ones_like(w))
        for call in (lambda: voc.token_logprobs(dual, t, top=1), lambda: voc.embed_tokens(dual, t), lambda: voc.clip_grad_norm_(dual, 1.0),
                     lambda: voc.embed_tokens_backward(dual, t, w, accumulate=False), lambda: voc.embed_tokens_backward(w, t, dual)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert bool((w == 1).all()) and bool((torch.autograd.forward_ad.unpack_dual(dual).primal == 1).all())
        assert torch.equal(voc.embed_tokens(w, t), w)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_the_norm_of_halves_keeps_small_numbers_beside_large_ones(voc, dtype):
    """1 and seven numbers whose squares, 2^-24, are half a step of it: added one after the other they vanish.  In 64 bits the sum of
    n such vectors is n (1 + 7 u); added by pairs, eight squares are off by three roundings at most, the norm by half of that and one
    rounding of its own: 2.5 u."""
    for n in (1, 67, 1059, 3000):
        g = torch.full((n, 8), 2.0 ** -12, device="cuda", dtype=dtype)
        g[:, 0] = 1
        want = math.sqrt(n * (1 + 7 * U))
        assert abs(float(voc.clip_grad_norm_([g], math.inf)) - want) <= 2.5 * U * (1 + 8 * U) * want


@gpu
@pytest.mark.parametrize("H", [7, 8])
@pytest.mark.parametrize("n", [6, 700])
@pytest.mark.parametrize("into", TYPES)
def test_embedding_gradient_beside_numbers_below_the_least_normal_one(voc, into, n, H):
    """Subnormal numbers of the table and of the gradient: kept in rows that do not occur, in a table that is overwritten, and in tables
    of halves.  What is added onto a float32 table may take each of the two operands and the result for 0."""
    least = torch.finfo(into).tiny
    t = torch.arange(n, device="cuda") % 3
    g = torch.zeros((n, H), device="cuda", dtype=into)
    g[0], g[1] = least / 4, least * 8  # token 0 below the least normal number, token 1 above
    table = torch.full((5, H), least / 2, device="cuda", dtype=into)
    more = table.clone()
    voc.embed_tokens_backward(g, t, more)
    want = table.double()
    want[0] += least / 4
    want[1] += least * 8
    assert torch.equal(more[3:], table[3:])  # no token of theirs: not touched
    if into == torch.float32:
        room = torch.full_like(want, 0.75 * least)  # all there is: least / 2 and least / 4, both taken for 0, or their sum
        room[1] = least / 2  # the table's; the result is a normal number
        _close(more, want, room)
    else:
        assert torch.equal(more.double(), want)
    d = voc.embed_tokens_backward(g, t, torch.empty_like(table), accumulate=False)
    want -= table.double()
    assert torch.equal(d.double(), want)


@gpu
@pytest.mark.parametrize("dtype, into", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("n", [0, 40, 256, 257, 6000])
@pytest.mark.parametrize("V", [1, 2, 3, 700, 150_000])
def test_embedding_gradient_into_columns_of_a_wider_table(voc, dtype, into, n, V):
    """Rows further apart than they are long, at any place of a 16-byte vector: what lies between them stays as it is."""
    gen = torch.Generator(device="cuda").manual_seed(V + n)
    for first, H, wide in ((8, 48, 64), (3, 48, 61), (1, 13, 16), (16, 8, 24), (0, 5, 7)):
        g = torch.randn((n, H), generator=gen, device="cuda").to(dtype)
        t = torch.randint(0, V, (n,), generator=gen, device="cuda")
        t[: n // 2] = V // 2
        want, room = _grad64(g, t, V, 1.5, 0)
        table = torch.full((V, wide), 7.0, device="cuda", dtype=into)
        part = table[:, first:first + H]
        part.fill_(math.nan)
        voc.embed_tokens_backward(g, t, part, scale=1.5, padding_idx=0, accumulate=False)
        _close(part, want, room, into)
        start = torch.randn((V, H), generator=gen, device="cuda").to(into)
        part.copy_(start)
        voc.embed_tokens_backward(g, t, part, scale=1.5, padding_idx=0)
        _close(part, want + start.double(), room + U * (want.abs() + start.double().abs()), into)
        assert bool((table[:, :first] == 7).all()) and bool((table[:, first + H:] == 7).all())


@gpu
def test_gradients_with_forward_mode_tangents_are_refused(voc):
    """The derivative of a gradient along a direction in which the incoming gradient changes: the kernels would drop it."""
    w = torch.randn((5, 3), device="cuda", requires_grad=True)
    t = torch.tensor([0, 4, 4, 1], device="cuda")
    with torch.autograd.forward_ad.dual_level():
        for shape, call in (((4, 3), lambda: voc.embed_tokens(w, t)), ((4,), lambda: voc.token_logprobs(w[:4], t.clamp(max=2)).logprob),
                            ((4, 2), lambda: voc.token_logprobs(w[:4], t.clamp(max=2), top=2).top_logprob),
                            ((4,), lambda: voc.token_logprobs(w[:4], t.clamp(max=2), entropy=True).entropy)):
            g = torch.randn(shape, device="cuda")
            dual = torch.autograd.forward_ad.make_dual(g, torch.ones_like(g))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad([call()], [w], [dual])
            d, = torch.autograd.grad([call()], [w], [g])  # without a tangent it goes on
            assert bool(d.isfinite().all())
