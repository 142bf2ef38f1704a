"""Performance cases of the vocabulary operators, through the public API.

Two operators: ``embed_tokens``, the lookup of rows of a shared table by token (Gaussians that hold
a token of a codebook, words of a query) with the table's gradient, and ``linear_cross_entropy``,
the softmax cross entropy of features (rendered pixels, words) against every row of a vocabulary
table, with the gradients of both.

A case is one pass: ``mode`` "eval" is the forward alone, "train" the forward and the gradients for
given upstream gradients.
"""

from __future__ import annotations

import math

import torch

own = False

IGNORED = -100
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _embed(name, count, vocab, dim, dtype, mode, tokens, *, index="int64", scale=1.0, padding=-1):
    """A lookup of ``count`` tokens in a (vocab, dim) table.  ``tokens``: their distribution:
    uniform, zipf (frequency about 1 / rank) or one (nine in ten are the same token);
    ``padding``: the padding token (-1: none)."""
    case = {"op": "embed", "count": count, "vocab": vocab, "dim": dim, "dtype": dtype, "mode": mode,
            "tokens": tokens, "index": index, "scale": scale, "padding": padding}
    return {"name": name, **case} if name else case


def _entropy(name, rows, vocab, dim, dtype, mode, *, reduction="mean", ignored=0.0, logit_scale=1.0, index="int64"):
    """A cross entropy of ``rows`` features over ``vocab`` classes; ``ignored``: the share of rows
    without a label."""
    case = {"op": "entropy", "rows": rows, "vocab": vocab, "dim": dim, "dtype": dtype, "mode": mode,
            "reduction": reduction, "ignored": ignored, "logit_scale": logit_scale, "index": index}
    return {"name": name, **case} if name else case


def listed():
    return [
        # One word of a query looked up: the smallest call, latency alone.
        _embed("lookup_1_d512", 1, 32768, 512, "bf16", "eval", "uniform", scale=math.sqrt(512.0)),
        # A scene of the benchmark's default size whose Gaussians hold tokens of a codebook.
        _embed("codebook_1m_d64", 1_000_000, 4096, 64, "fp32", "train", "zipf", index="int32"),
        # The largest scene's colour coefficients (degree 3: 16 x 3) from a codebook.
        _embed("codebook_5m_d48", 5_000_000, 8192, 48, "fp32", "train", "uniform", index="int32"),
        # A batch of text at the width of a text encoder, scaled as its features are.
        _embed("text_64k_d1024", 65536, 65536, 1024, "bf16", "train", "zipf", scale=32.0, padding=0),
        # Odd sizes, almost every position the same token (background), some padded.
        _embed("skewed_100k_d77", 100_003, 1203, 77, "fp16", "train", "one", padding=3),
        # One pixel's feature scored against the vocabulary: latency and one pass over the table.
        _entropy("score_1_v32k_d512", 1, 32768, 512, "bf16", "eval"),
        # A few picked pixels against a vocabulary of odd size, a loss for each.
        _entropy("score_37_v50001_d640", 37, 50001, 640, "fp16", "eval", reduction="none"),
        # An evaluation of one 256 x 256 image over a thousand classes: its map of losses.
        _entropy("image_64k_v1024_d256", 65536, 1024, 256, "bf16", "eval", reduction="none", ignored=0.1),
        # A training step on every pixel of an 800 x 800 image: rendered features in fp32, a small codebook.
        _entropy("pixels_640k_v512_d64", 640_000, 512, 64, "fp32", "train", ignored=0.2),
        # A training step on sampled pixels or words with a large vocabulary.
        _entropy("words_4k_v32k_d1024", 4096, 32768, 1024, "bf16", "train"),
        # A photograph of odd size (487 x 273), a vocabulary of odd size, weights for each pixel.
        _entropy("photo_133k_v1203_d100", 132_951, 1203, 100, "fp16", "train", reduction="none", ignored=0.3,
                 index="int32"),
        # The largest: a 256 x 256 image against a large vocabulary of joint text and image features.
        _entropy("image_64k_v32k_d512", 65536, 32768, 512, "bf16", "train", logit_scale=2.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    index = rng.choice(["int64", "int32"])
    mode = rng.choice(["eval", "train", "train"])
    if rng.random() < 0.4:
        dim = rng.choice([_log_int(rng, 1, 1024), 16 * _log_int(rng, 1, 64)])
        vocab = _log_int(rng, 16, 131072)
        count = _log_int(rng, 1, min(5_000_000, 240_000_000 // dim))
        return _embed(None, count, vocab, dim, dtype, mode, rng.choice(["uniform", "zipf", "one"]), index=index,
                      scale=rng.choice([1.0, math.sqrt(dim)]), padding=rng.choice([-1, -1, 0]))
    dim = rng.choice([_log_int(rng, 8, 1024), 64 * _log_int(rng, 1, 16)])
    vocab = rng.choice([_log_int(rng, 2, 65536), 2 ** rng.randint(6, 16)])
    # fp32 products cost about six times those of the 16-bit types
    budget = 65536 * 32768 * 512 // (6 if dtype == "fp32" else 1)
    most = max(1, min(640_000, budget // (vocab * dim), 2 ** 31 // vocab))
    return _entropy(None, _log_int(rng, 1, most), vocab, dim, dtype, mode,
                    reduction=rng.choice(["mean", "mean", "sum", "none"]), ignored=rng.choice([0.0, 0.1, 0.5]),
                    logit_scale=rng.choice([1.0, 1.0, 0.5, 3.0]), index=index)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _token_ids(case, gen):
    """Token positions of a case's distribution; the labels are shuffled, so that a frequent token is any row."""
    n, vocab = case["count"], case["vocab"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    if case["tokens"] == "zipf":
        rank = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    else:
        rank = (u * vocab).long().clamp_(0, vocab - 1)
    if case["tokens"] == "one":
        rank = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.9, torch.zeros_like(rank), rank)
    tokens = torch.randperm(vocab, generator=gen, device="cuda")[rank]
    if case["padding"] >= 0:
        tokens = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.05,
                             torch.full_like(tokens, case["padding"]), tokens)
    return tokens


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    index = torch.int32 if case["index"] == "int32" else torch.int64
    vocab, dim, train = case["vocab"], case["dim"], case["mode"] == "train"
    state = {"case": case}
    if case["op"] == "embed":
        state["tokens"] = _token_ids(case, gen).to(index)
        state["table"] = (_randn(gen, vocab, dim) / math.sqrt(dim)).to(dtype).requires_grad_(train)
        if train:
            state["upstream"] = _randn(gen, case["count"], dim).to(dtype)
        return state
    rows = case["rows"]
    table = (_randn(gen, vocab, dim) / math.sqrt(dim)).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    # a feature half way through a training: noise and a part along its label's row
    state["features"] = (_randn(gen, rows, dim) + 0.4 * math.sqrt(dim) * table[targets].float()).to(dtype)
    without = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
    state["targets"] = torch.where(without, torch.full_like(targets, IGNORED), targets).to(index)
    state["table"] = table.requires_grad_(train)
    state["features"].requires_grad_(train)
    if train:
        # a weight for each row, or the loss's own gradient
        state["upstream"] = (torch.rand(rows, generator=gen, device="cuda") + 0.5 if case["reduction"] == "none"
                             else torch.ones((), device="cuda"))
    return state


def _run_own(state):
    from gswarp_amd import vocabulary

    case = state["case"]
    if case["op"] == "embed":
        padding = None if case["padding"] < 0 else case["padding"]
        inputs = (state["table"],)

        def forward():
            return vocabulary.embed_tokens(state["tokens"], state["table"], scale=case["scale"], padding_idx=padding)
    else:
        inputs = (state["features"], state["table"])

        def forward():
            return vocabulary.linear_cross_entropy(
                state["features"], state["table"], state["targets"], ignore_index=IGNORED,
                reduction=case["reduction"], logit_scale=case["logit_scale"])

    if case["mode"] == "eval":
        with torch.no_grad():
            return [forward()]
    out = forward()
    grads = torch.autograd.grad(out, inputs, grad_outputs=state["upstream"])
    return [out.detach(), *grads]


def _plain_embed(state):
    case, table, tokens = state["case"], state["table"].detach().float(), state["tokens"].long()
    dtype = state["table"].dtype
    out = [(table[tokens] * case["scale"]).to(dtype)]
    if case["mode"] == "train":
        grad = torch.zeros_like(table)
        grad.index_add_(0, tokens, state["upstream"].float())
        if case["padding"] >= 0:
            grad[case["padding"]] = 0.0
        out.append((grad * case["scale"]).to(dtype))
    return out


def _plain_entropy(state):
    case = state["case"]
    features, table = state["features"].detach().float(), state["table"].detach().float()
    dtype, c = state["features"].dtype, case["logit_scale"]
    targets = state["targets"].long()
    valid = targets != IGNORED
    label = torch.where(valid, targets, torch.zeros_like(targets)).unsqueeze(1)
    logits = (features @ table.T) * c
    top = logits.amax(dim=1, keepdim=True)
    at_label = logits.gather(1, label).squeeze(1)
    share = logits.sub_(top).exp_()
    total = share.sum(dim=1, keepdim=True)
    loss = torch.where(valid, (total.log() + top).squeeze(1) - at_label, torch.zeros_like(at_label))
    count = valid.sum()
    reduced = {"none": lambda: loss, "sum": loss.sum, "mean": lambda: loss.sum() / count}[case["reduction"]]()
    if case["mode"] == "eval":
        return [reduced]
    weight = state["upstream"] / count if case["reduction"] == "mean" else state["upstream"]
    weight = torch.where(valid, weight.expand(valid.shape), torch.zeros_like(at_label))
    share /= total
    share.scatter_add_(1, label, torch.full_like(total, -1.0))
    share *= (weight * c).unsqueeze(1)
    return [reduced, (share @ table).to(dtype), (share.T @ features).to(dtype)]


def run(state):
    if own:
        return _run_own(state)
    return _plain_embed(state) if state["case"]["op"] == "embed" else _plain_entropy(state)


def exact(case, seed):
    """The definition in 64 bits."""
    state = prepare(case, seed)
    table = state["table"].detach().double()
    if case["op"] == "embed":
        tokens = state["tokens"].long()
        out = [torch.index_select(table, 0, tokens).mul_(case["scale"])]
        if case["mode"] == "train":
            kept = tokens != case["padding"]
            up = state["upstream"].double()[kept]
            out.append(torch.zeros_like(table).index_add_(0, tokens[kept], up, alpha=case["scale"]))
        return out
    features, targets = state["features"].detach().double(), state["targets"].long()
    rows, train, c = case["rows"], case["mode"] == "train", case["logit_scale"]
    kept = (targets != IGNORED).nonzero().squeeze(1)
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    grad_features, grad_table = torch.zeros_like(features), torch.zeros_like(table)
    piece = max(1, 2 ** 28 // case["vocab"])
    for ids in kept.split(piece):
        h, t = features[ids], targets[ids]
        s = c * torch.matmul(h, table.T)
        log_p = s - torch.logsumexp(s, dim=1, keepdim=True)
        at = torch.arange(ids.numel(), device="cuda")
        loss[ids] = -log_p[at, t]
        if train:
            ds = log_p.exp()
            ds[at, t] -= 1.0
            w = state["upstream"].double()
            w = w[ids] if case["reduction"] == "none" else w / (kept.numel() if case["reduction"] == "mean" else 1)
            ds *= c * (w.unsqueeze(1) if w.ndim else w)
            grad_features[ids] = torch.matmul(ds, table)
            grad_table += torch.matmul(ds.T.contiguous(), h)
    if case["reduction"] != "none":
        loss = loss.sum() / (kept.numel() if case["reduction"] == "mean" else 1)
    return [loss, grad_features, grad_table] if train else [loss]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    index = 4 if case["index"] == "int32" else 8
    train, vocab, dim = case["mode"] == "train", case["vocab"], case["dim"]
    if case["op"] == "embed":
        n = case["count"]
        moved = n * index + min(n, vocab) * dim * size + n * dim * size
        if train:
            moved += n * dim * size + vocab * dim * size
        return {"bytes": moved, "flops": n * dim * (2 if train else 1)}
    rows = case["rows"]
    labelled = rows * (1.0 - case["ignored"])
    moved = rows * index + (labelled + vocab) * dim * size + (rows * 4 if case["reduction"] == "none" else 4)
    if train:
        moved += (rows + vocab) * dim * size + (rows * 4 if case["reduction"] == "none" else 4)
    # the logits, and their products with the table and the features
    return {"bytes": int(moved), "flops": int((6 if train else 2) * labelled * vocab * dim)}
