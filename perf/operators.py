"""The operators at both ends of the vocabulary table and behind the backward pass, with their inputs and work.

A case's ``op`` says which of them it calls:

* ``logprobs`` — log probabilities of given tokens from materialised logits, with entropy and the ``top`` best
  alternatives; ``grad``: as a training step, with the gradient of the logits;
* ``embed``    — embedding lookup with scaling; ``grad``: with the table's gradient, dense, in the table's type;
* ``tied``     — the embedding's gradient added onto the output projection's float32 weight gradient (shared table);
* ``clip``     — global norm of a model's gradients and clipping, in place or into float32 master gradients.

Rows behind a sentence's end hold the padding token: they are left out of the log probabilities and of the table's gradient.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

PAD, UNK = 1, 3
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}


def _operators():
    """The package of the repository that the program runs in (its directory's name is not an identifier)."""
    name = "pcfg_nat_b200"
    if name not in sys.modules:
        home = os.path.join(os.getcwd(), "pcfg-nat_b200")
        home = home if os.path.isdir(home) else os.path.join(ROOT, "pcfg-nat_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(home, "__init__.py"),
                                                      submodule_search_locations=[home])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module("pcfg_nat_b200.custom_ops")


def _logprobs(name, batch, shortest, longest, vocab, dtype, top=0, grad=False, pitch=0):
    return dict(name=name, op="logprobs", batch=batch, shortest=shortest, longest=longest, vocab=vocab, dtype=dtype, top=top,
                grad=grad, pitch=pitch or vocab)


def _embed(name, op, batch, shortest, longest, vocab, hidden, dtype, grad, unknown):
    return dict(name=name, op=op, batch=batch, shortest=shortest, longest=longest, vocab=vocab, hidden=hidden, dtype=dtype,
                grad=grad, unknown=unknown)


def _clip(name, layers, vocab, hidden, dtype, into, clipped):
    return dict(name=name, op="clip", layers=layers, vocab=vocab, hidden=hidden, dtype=dtype, into=into, clipped=clipped)


def listed():
    return [
        # the answer to one request, with the alternatives that a confidence display shows: latency
        _logprobs("score_one", 1, 33, 33, 40000, "float16", top=5),
        # a batch of candidate answers of mixed lengths, scored for reranking
        _logprobs("score_batch", 64, 10, 61, 40000, "bfloat16", top=8),
        # a training batch on the decoder's graph: likelihood with an entropy term, half precision
        _logprobs("train_batch", 90, 80, 160, 40000, "float16", grad=True),
        # a dictionary that is no multiple of anything, single precision, target side only
        _logprobs("train_odd", 45, 20, 40, 39999, "float32", grad=True),
        # decoder input of one sentence: latency
        _embed("embed_one", "embed", 1, 140, 140, 40000, 512, "float16", False, 0.0),
        # decoder input of a glancing pass: most nodes hold the placeholder, the rest revealed words
        _embed("embed_glancing", "embed", 90, 80, 160, 40000, 512, "float16", True, 0.7),
        # text of the usual word frequencies, single precision, rows that are no multiple of 16 bytes
        _embed("embed_text", "embed", 128, 64, 256, 32001, 301, "float32", True, 0.0),
        # the gradient of the shared table: the decoder input's on the model's graph, added onto the projection's
        _embed("tied_graph", "tied", 90, 162, 322, 40000, 512, "float16", True, 0.7),
        # a toy model's gradients, copied out as an optimizer with its own buffers wants them: launches and latency
        _clip("clip_toy", 1, 1000, 64, "float32", "float32", True),
        # a base model's half-precision gradients, loss scale taken out, clipped into float32 master gradients
        _clip("clip_master", 6, 40000, 512, "float16", "float32", True),
        # the same model in single precision, in place, below the limit: the norm is all that is asked for
        _clip("clip_quiet", 6, 40000, 512, "float32", "itself", False),
    ]


def draw(rng):
    log_int = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["logprobs", "logprobs", "logprobs", "embed", "embed", "tied", "clip"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    longest = log_int(1, 322)
    batch = log_int(1, max(1, min(128, 14000 // longest)))
    shortest = max(1, int(longest * rng.uniform(0.2, 1.0)))
    vocab = log_int(500, 40000)
    if op == "logprobs":
        grad = rng.random() < 0.5
        if dtype == "float32":
            batch = max(1, batch // 2)
        return dict(op=op, batch=batch, shortest=shortest, longest=longest, vocab=vocab, dtype=dtype, top=0 if grad else rng.choice([0, 1, 5, 20]),
                    grad=grad, pitch=rng.choice([vocab, (vocab + 63) // 64 * 64]))
    if op in ("embed", "tied"):
        return dict(op=op, batch=batch, shortest=shortest, longest=longest, vocab=vocab, dtype=dtype,
                    hidden=rng.choice([64, 128, 256, 512, 512, log_int(33, 700)]), grad=op == "tied" or rng.random() < 0.6,
                    unknown=rng.choice([0.0, 0.3, 0.7, 0.9]))
    into = rng.choice(["itself", "float32"])
    # what is clipped in place is below the limit from the second pass on: such a case would not be the same twice
    return dict(op=op, layers=rng.randint(1, 6), vocab=vocab, hidden=rng.choice([64, 128, 256, 512, log_int(33, 500)]), dtype=dtype,
                into=into, clipped=into == "float32" and rng.random() < 0.7)


def _lengths(case):
    B, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi - (hi - lo) * i // max(1, B - 1) for i in range(B)]


def _shapes(case):
    """The tensors of an encoder and decoder of ``layers`` layers each, with the shared table first."""
    d, f = case["hidden"], 4 * case["hidden"]
    attention = [(d, d), (d,)] * 4 + [(d,), (d,)]
    layer = [(f, d), (f,), (d, f), (d,), (d,), (d,)]
    return [(case["vocab"], d)] + (2 * case["layers"]) * (attention + layer) + case["layers"] * attention + [(d,), (d,)]


def _count(case):
    return sum(math.prod(s) for s in _shapes(case))


def _tokens(g, case, dev):
    """[B, L] with padding behind every sentence, words by the usual law of frequencies, placeholders among them."""
    B, L, V = case["batch"], case["longest"], case["vocab"]
    lengths = torch.tensor(_lengths(case), device=dev)
    words = 4 + (torch.rand((B, L), generator=g, device=dev) * math.log(V - 4)).exp().floor().long().clamp_(max=V - 5)
    unknown = torch.rand((B, L), generator=g, device=dev) < case.get("unknown", 0.0)
    words = torch.where(unknown, UNK, words)
    return torch.where(torch.arange(L, device=dev)[None] < lengths[:, None], words, PAD)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case, op=case["op"])
    dtype = TYPES[case["dtype"]]
    if case["op"] == "clip":
        n, shapes = _count(case), _shapes(case)
        flat = torch.randn(n, generator=g, device=dev)
        flat *= 0.001 * (1 << 7 if dtype == torch.float16 else 1)  # half-precision gradients carry a loss scale
        flat = flat.to(dtype)
        s["scale"] = 1.0 / (1 << 7) if dtype == torch.float16 else 1.0
        s["max_norm"] = (0.3 if case["clipped"] else 3.0) * 0.001 * math.sqrt(n)
        s["flat"], s["grads"] = flat, [v.view(d) for v, d in zip(flat.split([math.prod(d) for d in shapes]), shapes)]
        s["flat_out"] = torch.empty(n, device=dev) if case["into"] == "float32" else flat
        s["out"] = [v.view(d) for v, d in zip(s["flat_out"].split([math.prod(d) for d in shapes]), shapes)]
        return s
    tokens = _tokens(g, case, dev)
    s["tokens"] = tokens
    if case["op"] == "logprobs":
        x = torch.empty(tokens.shape + (case["pitch"],), device=dev, dtype=dtype)
        for b in range(case["batch"]):  # a sentence at a time: the float32 numbers need not all be there at once
            row = torch.randn((case["longest"], case["pitch"]), generator=g, device=dev) * 2
            lift = torch.rand((case["longest"], 1), generator=g, device=dev) * 14  # from hardly trained to confident
            x[b] = row.scatter_add_(1, tokens[b][:, None], lift).to(dtype)
        s["logits"] = x[..., :case["vocab"]]
        if case["grad"]:
            s["logits"].requires_grad_(True)
            s["g_logprob"] = -torch.rand(tokens.shape, generator=g, device=dev) - 0.5
            s["g_entropy"] = torch.full(tokens.shape, -0.01, device=dev)
        return s
    V, H = case["vocab"], case["hidden"]
    s["scale"] = math.sqrt(H)
    if case["op"] == "embed":
        s["weight"] = (torch.randn((V, H), generator=g, device=dev) / math.sqrt(H)).to(dtype).requires_grad_(case["grad"])
    else:
        s["d_weight"] = torch.randn((V, H), generator=g, device=dev)
    if case["grad"]:
        s["g_out"] = torch.randn(tokens.shape + (H,), generator=g, device=dev).to(dtype)
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"logprobs": _plain_logprobs, "embed": _plain_embed, "tied": _plain_tied, "clip": _plain_clip}[s["op"]](s)


def _run_own(s):
    ops, case = _operators(), s["case"]
    if s["op"] == "clip":
        norm = ops.clip_grad_norm_(s["grads"], s["max_norm"], out=s["out"] if case["into"] == "float32" else None,
                                   grad_scale=s["scale"])
        return {"norm": norm, "clipped": s["flat_out"]}
    if s["op"] == "logprobs":
        got = ops.token_logprobs(s["logits"], s["tokens"], top=case["top"], entropy=True, ignore_index=PAD)
        out = {"logprob": got.logprob, "entropy": got.entropy}
        if case["top"]:
            out["top_logprob"], out["top_index"] = got.top_logprob, got.top_index
        if case["grad"]:
            out["d_logits"], = torch.autograd.grad([got.logprob, got.entropy], [s["logits"]], [s["g_logprob"], s["g_entropy"]])
        return out
    if s["op"] == "tied":
        return {"d_weight": ops.embed_tokens_backward(s["g_out"], s["tokens"], s["d_weight"], scale=s["scale"], padding_idx=PAD)}
    out = ops.embed_tokens(s["weight"], s["tokens"], scale=s["scale"], padding_idx=PAD)
    if not case["grad"]:
        return {"out": out}
    d_weight, = torch.autograd.grad([out], [s["weight"]], [s["g_out"]])
    return {"out": out, "d_weight": d_weight}


def _plain_logprobs(s):
    case, tokens, x = s["case"], s["tokens"], s["logits"].detach()
    dtype, x = x.dtype, x.float()
    keep = tokens != PAD
    y = x - x.amax(-1, keepdim=True)
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    lp = y - total.log()
    p = e / total
    entropy = -(p * lp).sum(-1)
    logprob = lp.gather(-1, tokens[..., None])[..., 0]
    out = {"logprob": torch.where(keep, logprob, 0.0), "entropy": torch.where(keep, entropy, 0.0)}
    if case["top"]:
        # whole numbers in the order of the values, equal ones by falling index
        bits = (x + 0.0).view(torch.int32)
        rank = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + ((1 << 32) - 1 - torch.arange(x.shape[-1], device=x.device))
        index = (1 << 32) - 1 - (rank.topk(case["top"], -1).values & 0xFFFFFFFF)
        out["top_logprob"] = torch.where(keep[..., None], lp.gather(-1, index), 0.0)
        out["top_index"] = torch.where(keep[..., None], index, -1)
    if case["grad"]:
        g, h = s["g_logprob"][..., None], s["g_entropy"][..., None]
        d = -p * (g + h * (lp + entropy[..., None]))
        d.scatter_add_(-1, tokens[..., None], g)
        out["d_logits"] = torch.where(keep[..., None], d, 0.0).to(dtype)
    return out


def _plain_embed(s):
    case, tokens, weight = s["case"], s["tokens"], s["weight"].detach()
    out = {"out": (weight[tokens].float() * s["scale"]).to(weight.dtype)}
    if case["grad"]:
        g = torch.where((tokens != PAD)[..., None], s["g_out"].float() * s["scale"], 0.0)
        d = torch.zeros(weight.shape, device=weight.device)
        out["d_weight"] = d.index_add_(0, tokens.flatten(), g.flatten(0, 1)).to(weight.dtype)
    return out


def _plain_tied(s):
    tokens = s["tokens"]
    g = torch.where((tokens != PAD)[..., None], s["g_out"].float() * s["scale"], 0.0)
    return {"d_weight": s["d_weight"].index_add_(0, tokens.flatten(), g.flatten(0, 1))}


def _plain_clip(s):
    squares = torch.stack([(g.float() * s["scale"]).square().sum() for g in s["grads"]])
    norm = squares.sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0) * s["scale"]
    [o.copy_(g.float() * factor) for o, g in zip(s["out"], s["grads"])]
    return {"norm": norm, "clipped": s["flat_out"]}


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "clip":
        n = _count(case)
        back = n * (4 if case["into"] == "float32" else size if case["clipped"] else 0)
        return {"bytes": n * size + back, "flops": 3 * n}
    rows, real = case["batch"] * case["longest"], sum(_lengths(case))
    if case["op"] == "logprobs":
        n, V = real, case["vocab"]
        once = n * V * size + rows * (16 + 12 * case["top"])
        if not case["grad"]:
            return {"bytes": once, "flops": 6 * n * V}
        return {"bytes": once + rows * V * size + 8 * rows, "flops": 11 * n * V}  # the logits are read once, their gradient is written
    H, V = case["hidden"], case["vocab"]
    words = min(V, real)  # at most that many rows of the table are touched; placeholders share one
    words = max(1, min(words, int(real * (1 - case["unknown"])) + 1))
    if case["op"] == "tied":
        return {"bytes": real * H * size + rows * 8 + 8 * words * H, "flops": 2 * real * H}
    there = rows * 8 + words * H * size + rows * H * size
    if not case["grad"]:
        return {"bytes": there, "flops": rows * H}
    return {"bytes": there + real * H * size + V * H * size, "flops": 3 * rows * H}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        x = s["flat"].double() * s["scale"]
        norm = torch.linalg.vector_norm(x)
        return {"norm": norm, "clipped": x * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}
    tokens = s["tokens"]
    keep = tokens.ne(PAD)
    if case["op"] == "logprobs":
        got = {k: [] for k in ("logprob", "entropy", "top_logprob", "d_logits")}
        for b in range(case["batch"]):
            z = s["logits"][b].detach().double()
            lp = torch.log_softmax(z, -1)
            p, on = lp.exp(), keep[b][:, None].double()
            H = -(p * lp).sum(-1, keepdim=True)
            hot = torch.zeros_like(lp)
            hot[torch.arange(len(z), device=z.device), tokens[b]] = 1.0
            got["logprob"].append((on * hot * lp).sum(-1))
            got["entropy"].append((on * H)[:, 0])
            if case["top"]:
                got["top_logprob"].append(on * lp.topk(case["top"], -1).values)
            if case["grad"]:
                u, v = s["g_logprob"][b][:, None].double(), s["g_entropy"][b][:, None].double()
                got["d_logits"].append((on * (u * (hot - p) - v * p * (lp + H))).float())  # 64 bits until here: a fraction of the memory
        return {k: torch.stack(v) for k, v in got.items() if v}
    V, H = case["vocab"], case["hidden"]
    out = {}
    if case["op"] == "embed":
        out["out"] = torch.nn.functional.embedding(tokens, s["weight"].detach().double()) * s["scale"]
    if case["grad"]:
        at, order = tokens.flatten()[keep.flatten()].sort(stable=True)
        terms = s["g_out"].flatten(0, 1)[keep.flatten()][order].double() * s["scale"]
        d = torch.zeros((V, H), device=terms.device, dtype=torch.float64).index_put_((at,), terms, accumulate=True)
        out["d_weight"] = d + s["d_weight"].double() if case["op"] == "tied" else d
    return out
