"""embed_tokens and linear_cross_entropy against their definitions in 64 bits, at the sizes, masks,
strides and values where they can go wrong."""

from __future__ import annotations

import math

import pytest
import torch

from gswarp_amd import vocabulary
import vocabulary_ref as ref

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = [FP32, BF16, FP16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tokens(kind, n, vocab, gen):
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=gen)
    if kind == "one":
        return torch.full((n,), vocab // 2)
    if kind == "sorted":
        return torch.randint(0, vocab, (n,), generator=gen).sort().values
    # zipf: about 1 / rank
    return (torch.exp(torch.rand(n, generator=gen, dtype=torch.float64) * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1)


# ---------------------------------------------------------------- lookup

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,dim,kind", [
    (1, 1, 1, "uniform"), (1, 300, 64, "uniform"), (2, 5, 3, "one"), (7, 2, 130, "uniform"), (63, 1000, 8, "zipf"),
    (64, 64, 16, "sorted"), (65, 3, 77, "zipf"), (255, 4096, 48, "uniform"), (1025, 33, 1024, "zipf"),
    (4099, 5000, 2, "uniform"), (5000, 7, 45, "one"), (20011, 513, 24, "zipf"), (70001, 31, 12, "one"),
    (9973, 128, 1037, "zipf"), (300_007, 100, 4, "uniform")])
def test_lookup_and_gradient(device, dtype, n, vocab, dim, kind):
    print(f"lookup {dtype} n={n} vocab={vocab} dim={dim} {kind}", flush=True)
    gen = _gen(n + dim)
    tokens = _tokens(kind, n, vocab, gen).to(device, torch.int32 if n % 2 else torch.int64)
    table = torch.randn(vocab, dim, generator=gen).to(device, dtype).requires_grad_(True)
    up = torch.randn(n, dim, generator=gen).to(device, dtype)
    padding = None if n % 3 else 0
    for scale in (1.0, 2.7):
        out = vocabulary.embed_tokens(tokens, table, scale=scale, padding_idx=padding)
        assert out.dtype == dtype and out.shape == (n, dim)
        ref.check(out, ref.embed(tokens, table.detach(), scale), "out")
        (grad,) = torch.autograd.grad(out, table, up)
        assert grad.dtype == dtype
        ref.check(grad, ref.embed_grad(tokens, up, vocab, scale, padding), "grad")
        (again,) = torch.autograd.grad(vocabulary.embed_tokens(tokens, table, scale=scale, padding_idx=padding),
                                       table, up)
        assert torch.equal(grad, again)


def test_lookup_shapes_and_no_positions(device):
    table = torch.randn(9, 20, device=device, requires_grad=True)
    assert vocabulary.embed_tokens(torch.tensor(4, device=device), table).shape == (20,)
    assert vocabulary.embed_tokens(torch.zeros(2, 3, dtype=torch.int32, device=device), table).shape == (2, 3, 20)
    out = vocabulary.embed_tokens(torch.empty(0, 5, dtype=torch.int64, device=device), table)
    assert out.shape == (0, 5, 20)
    (grad,) = torch.autograd.grad(out, table, torch.empty_like(out))
    assert torch.equal(grad, torch.zeros_like(table))


def test_lookup_outside_the_table(device):
    """Rows of NaN, no read and no gradient; int64 values that 32 bits would wrap into the table included."""
    table = torch.randn(6, 10, device=device, requires_grad=True)
    tokens = torch.tensor([0, -1, 6, 2 ** 32 + 1, -2 ** 63, 2 ** 63 - 1, 5], device=device)
    out = vocabulary.embed_tokens(tokens, table)
    bad = torch.tensor([False, True, True, True, True, True, False], device=device)
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], table[tokens[~bad]])
    up = torch.randn(7, 10, device=device)
    (grad,) = torch.autograd.grad(out, table, up)
    ref.check(grad, ref.embed_grad(tokens, up, 6, 1.0), "grad")


def test_lookup_padding_ignores_its_gradient(device):
    """Infinities and NaN at padded positions do not reach the gradient."""
    table = torch.randn(5, 33, device=device, requires_grad=True)
    tokens = torch.tensor([1, 2, 2, 4, 2, 1], device=device)
    out = vocabulary.embed_tokens(tokens, table, padding_idx=2)
    assert torch.equal(out, table[tokens])
    up = torch.randn(6, 33, device=device)
    up[tokens == 2] = math.nan
    up[2] = math.inf
    (grad,) = torch.autograd.grad(out, table, up)
    ref.check(grad, ref.embed_grad(tokens, up, 5, 1.0, padding=2), "grad")
    tokens = torch.full((1000,), 2, device=device)  # nothing left
    (grad,) = torch.autograd.grad(vocabulary.embed_tokens(tokens, table, padding_idx=2), table,
                                  torch.full((1000, 33), math.nan, device=device))
    assert torch.equal(grad, torch.zeros_like(table))


@pytest.mark.parametrize("dtype", DTYPES)
def test_lookup_strided_and_unaligned(device, dtype):
    gen = _gen(3)
    wide = torch.randn(50, 200, generator=gen).to(device, dtype)
    tokens = torch.randint(0, 50, (2, 700), generator=gen).to(device)
    strided = tokens.T  # (700, 2), not contiguous
    for table in (wide[:, 8:72], wide[:, 3:67], wide[:, 1:14], wide[::2].repeat(2, 1)[:, :64], wide.T[:50, :50],
                  wide[:1].expand(50, 200)):
        leaf = table.detach().requires_grad_(True)
        out = vocabulary.embed_tokens(strided, leaf)
        assert torch.equal(out, table[strided])
        up = torch.randn(out.shape[0], out.shape[1], 2 * out.shape[2], generator=gen).to(device, dtype)[..., ::2]
        (grad,) = torch.autograd.grad(out, leaf, up)
        ref.check(grad, ref.embed_grad(strided, up, 50, 1.0), "grad")


def test_lookup_past_32_bits(device):
    """A table and an output whose byte offsets pass 2^32 and whose element offsets pass 2^31."""
    vocab, dim = 1_100_000, 2048
    table = torch.zeros(vocab, dim, dtype=BF16, device=device)
    rows = torch.tensor([0, 1, vocab // 2, vocab - 2, vocab - 1], device=device)
    table[rows] = torch.randn(5, dim, generator=_gen(1)).to(device, BF16)
    tokens = torch.full((vocab,), 7, dtype=torch.int32, device=device)
    tokens[-5:] = rows.int()
    out = vocabulary.embed_tokens(tokens, table)
    assert torch.equal(out[-5:], table[rows]) and not out[:-5].any()
    del out
    leaf = table.requires_grad_(True)
    up = torch.zeros(vocab, dim, dtype=BF16, device=device)
    up[-5:] = 1.0
    up[5] = 3.0
    (grad,) = torch.autograd.grad(vocabulary.embed_tokens(tokens, leaf), leaf, up)
    want = torch.ones(5, dim, dtype=BF16, device=device)
    assert torch.equal(grad[rows], want) and bool((grad[7] == 3.0).all())
    grad[rows] = 0
    grad[7] = 0
    assert not grad.any()


# ---------------------------------------------------------------- cross entropy

def _problem(device, dtype, rows, vocab, dim, seed=0, ignored=0.2, spread=1.0):
    gen = _gen(seed + rows * 7 + vocab + dim)
    features = (torch.randn(rows, dim, generator=gen) * spread).to(device, dtype)
    table = (torch.randn(vocab, dim, generator=gen) / math.sqrt(dim)).to(device, dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen)
    targets[torch.rand(rows, generator=gen) < ignored] = -100
    return features.requires_grad_(True), table.requires_grad_(True), targets.to(device), gen


def _compare(features, table, targets, upstream, **options):
    loss = vocabulary.linear_cross_entropy(features, table, targets, **options)
    with torch.no_grad():
        alone = vocabulary.linear_cross_entropy(features, table, targets, **options)
    want = ref.entropy(features.detach(), table.detach(), targets, upstream, **options)
    assert loss.dtype == FP32
    ref.check(loss, want["loss"], "loss")
    ref.check(alone, want["loss"], "loss without a gradient")
    grads = torch.autograd.grad(loss, (features, table), upstream)
    for name, got in zip(("features", "table"), grads):
        assert got.dtype == table.dtype
        ref.check(got, want[name], name)
    return loss, grads


SIZES = [(1, 1, 1), (1, 2, 8), (3, 5, 7), (2, 300, 16), (16, 1000, 40), (17, 129, 64), (33, 64, 65), (64, 128, 64),
         (65, 130, 72), (127, 127, 128), (129, 257, 200), (300, 70, 33), (257, 1203, 100), (1000, 513, 24),
         (40, 5000, 264), (5000, 40, 136), (700, 600, 520)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", SIZES)
def test_entropy(device, dtype, rows, vocab, dim):
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim}", flush=True)
    features, table, targets, gen = _problem(device, dtype, rows, vocab, dim)
    if not bool((targets != -100).any()):
        targets[0] = 0
    if rows % 2:
        targets = targets.int()
    for reduction in ("mean", "sum", "none"):
        up = (torch.rand(rows, generator=gen) + 0.5).to(device) if reduction == "none" else torch.tensor(0.7, device=device)
        first = _compare(features, table, targets, up, reduction=reduction, logit_scale=1.5)
        loss = vocabulary.linear_cross_entropy(features, table, targets, reduction=reduction, logit_scale=1.5)
        grads = torch.autograd.grad(loss, (features, table), up)
        assert torch.equal(loss, first[0]) and all(torch.equal(a, b) for a, b in zip(grads, first[1]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("logit_scale", [0.0, -2.0, 30.0])
def test_entropy_scales(device, dtype, logit_scale):
    """A flat, an inverted and an almost certain distribution."""
    features, table, targets, gen = _problem(device, dtype, 200, 333, 48)
    _compare(features, table, targets, torch.tensor(1.0, device=device), logit_scale=logit_scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(200, 1, 16), (200, 2, 16), (300, 3, 128), (100, 65, 24), (90, 67, 256),
                                            (70, 66, 192), (600, 700, 64), (513, 1025, 60), (66, 5, 130), (1, 900, 64)])
def test_entropy_few_classes_and_short_rows(device, dtype, rows, vocab, dim):
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim}", flush=True)
    features, table, targets, gen = _problem(device, dtype, rows, vocab, dim, ignored=0.1 if rows > 1 else 0.0)
    for reduction, logit_scale in (("mean", 1.0), ("none", -1.5)):
        up = torch.rand(rows, generator=gen).to(device) if reduction == "none" else torch.tensor(1.0, device=device)
        _compare(features, table, targets, up, reduction=reduction, logit_scale=logit_scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,dim", [(3, 100, 64), (200, 100, 64), (200, 300, 128), (200, 300, 320)])
def test_entropy_of_certain_labels(device, dtype, rows, vocab, dim):
    """Labels of all but probability 1 (everything else together below 2^-26): the largest of a
    row counts as exactly 1, so a loss and a gradient may be lost, but nothing larger takes their place."""
    gen = _gen(rows + dim)
    table = (torch.randn(vocab, dim, generator=gen) / math.sqrt(dim)).to(device, dtype)
    targets = torch.randint(0, vocab, (rows,), generator=gen).to(device)
    h = 60.0 * table[targets].float() / table[targets].float().square().sum(1, keepdim=True)
    features = h.to(dtype).requires_grad_(True)
    leaf = table.clone().requires_grad_(True)
    loss = vocabulary.linear_cross_entropy(features, leaf, targets, reduction="none", logit_scale=1.3)
    s = 1.3 * (features.detach().double() @ table.double().T)
    rest = torch.softmax(s, 1)
    rest[torch.arange(rows, device=device), targets] = 0.0
    rest = rest.sum(1)
    assert float(rest.max()) < 2.0 ** -26
    exact = torch.log1p(rest)
    assert bool((loss >= 0).all()) and bool(((loss.double() - exact).abs() <= exact * 1.01).all())
    grads = torch.autograd.grad(loss, (features, leaf), torch.ones_like(loss))
    # each row's ds has 1-norm 2 rest
    bound = 1.3 * 2 * rest.unsqueeze(1) * table.double().abs().amax() * 1.01 + ref.TINY[dtype]
    assert bool((grads[0].double().abs() <= bound).all())
    bound = 1.3 * 2 * rest.sum() * features.detach().double().abs().amax() * 1.01 + ref.TINY[dtype]
    assert bool((grads[1].double().abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_entropy_ignored_rows_hold_anything(device, dtype):
    """NaN, infinities and the type's largest values in rows that do not count."""
    features, table, targets, gen = _problem(device, dtype, 333, 150, 72, ignored=0.4)
    hostile = features.detach().clone()
    gone = (targets == -100).nonzero().squeeze(1)
    fill = [math.nan, math.inf, -math.inf, torch.finfo(dtype).max, torch.finfo(dtype).min]
    for i, row in enumerate(gone.tolist()):
        hostile[row] = fill[i % 5]
    hostile.requires_grad_(True)
    for reduction in ("mean", "none"):
        up = torch.ones(333 if reduction == "none" else (), device=device)
        hostile_up = up.clone()
        if reduction == "none":
            hostile_up[gone] = math.nan
        got = vocabulary.linear_cross_entropy(hostile, table, targets, reduction=reduction)
        base = vocabulary.linear_cross_entropy(features, table, targets, reduction=reduction)
        assert torch.equal(got, base)
        mine = torch.autograd.grad(got, (hostile, table), hostile_up)
        theirs = torch.autograd.grad(base, (features, table), up)
        assert all(torch.equal(a, b) for a, b in zip(mine, theirs))
        assert not mine[0][gone].any()


def test_entropy_nothing_counts(device):
    features, table, targets, _ = _problem(device, BF16, 150, 300, 64)
    targets.fill_(-100)
    loss = vocabulary.linear_cross_entropy(features, table, targets)
    assert torch.isnan(loss)  # the mean over nothing
    for reduction in ("mean", "sum", "none"):
        loss = vocabulary.linear_cross_entropy(features, table, targets, reduction=reduction)
        if reduction != "mean":
            assert not loss.any()
        for grad in torch.autograd.grad(loss, (features, table), torch.ones_like(loss)):
            assert torch.equal(grad, torch.zeros_like(grad))


def test_entropy_no_rows(device):
    table = torch.randn(40, 24, device=device, requires_grad=True)
    features = torch.empty(0, 24, device=device, requires_grad=True)
    targets = torch.empty(0, dtype=torch.int64, device=device)
    assert vocabulary.linear_cross_entropy(features, table, targets, reduction="none").shape == (0,)
    assert vocabulary.linear_cross_entropy(features, table, targets, reduction="sum").item() == 0.0
    loss = vocabulary.linear_cross_entropy(features, table, targets)
    assert torch.isnan(loss)
    grads = torch.autograd.grad(loss, (features, table))
    assert grads[0].shape == (0, 24) and torch.equal(grads[1], torch.zeros_like(table))


def test_entropy_another_ignore_index_and_shapes(device):
    features, table, targets, _ = _problem(device, FP16, 60, 90, 32, ignored=0.0)
    targets[::7] = 5
    grid, grid_targets = features.detach().reshape(3, 20, 32).requires_grad_(True), targets.reshape(3, 20)
    loss = vocabulary.linear_cross_entropy(grid, table, grid_targets, ignore_index=5, reduction="none")
    assert loss.shape == (3, 20) and not loss[grid_targets == 5].any()
    want = ref.entropy(features.detach(), table.detach(), targets, torch.ones(60, device=device), ignore_index=5,
                       reduction="none")
    ref.check(loss, want["loss"], "loss")
    grads = torch.autograd.grad(loss, (grid, table), torch.ones_like(loss))
    assert grads[0].shape == (3, 20, 32)
    ref.check(grads[0], want["features"], "features")
    ref.check(grads[1], want["table"], "table")
    one = vocabulary.linear_cross_entropy(grid[0, 1].detach(), table.detach(), grid_targets[0, 1], reduction="none")
    assert one.shape == ()


def test_entropy_targets_outside_the_vocabulary(device):
    """NaN for their rows alone; int64 values that 32 bits would wrap into the vocabulary included."""
    features, table, targets, _ = _problem(device, FP32, 50, 70, 32, ignored=0.0)
    base = vocabulary.linear_cross_entropy(features, table, targets, reduction="none")
    bad = targets.clone()
    bad[3], bad[10], bad[11], bad[12] = -1, 70, 2 ** 32 + 3, -2 ** 63
    loss = vocabulary.linear_cross_entropy(features, table, bad, reduction="none")
    is_bad = torch.zeros(50, dtype=torch.bool, device=device)
    is_bad[[3, 10, 11, 12]] = True
    assert torch.isnan(loss[is_bad]).all() and torch.equal(loss[~is_bad], base[~is_bad])
    assert torch.isnan(vocabulary.linear_cross_entropy(features, table, bad))
    (grad,) = torch.autograd.grad(loss, features, torch.ones_like(loss))
    assert torch.isnan(grad[is_bad]).all() and torch.isfinite(grad[~is_bad]).all()


def test_entropy_non_finite_rows_stay_alone(device):
    features, table, targets, _ = _problem(device, BF16, 200, 300, 64, ignored=0.0)
    bad = features.detach().clone()
    bad[17, 3] = math.nan
    bad[90, 5] = math.inf
    got = vocabulary.linear_cross_entropy(bad, table.detach(), targets, reduction="none")
    want = vocabulary.linear_cross_entropy(features.detach(), table.detach(), targets, reduction="none")
    keep = torch.ones(200, dtype=torch.bool, device=device)
    keep[[17, 90]] = False
    assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[~keep]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_entropy_strided_and_unaligned(device, dtype):
    gen = _gen(11)
    wide = torch.randn(120, 400, generator=gen).to(device, dtype)
    targets = torch.randint(0, 50, (70,), generator=gen).to(device)
    for f, t in ((wide[:70, :64], wide[70:, 64:128]), (wide[:70, 1:65], wide[70:, 3:67]), (wide[:70, :65], wide[70:, 5:70]),
                 (wide[:70].T[:70, :33], wide.T[100:150, :33]), (wide[::1][:70, ::4], wide[70:, 1::4]),
                 (wide[:1, :40].expand(70, 40), wide[70:, :40])):
        features, table = f.detach().requires_grad_(True), (t.detach() / 8).requires_grad_(True)
        _compare(features, table, targets, torch.tensor(1.0, device=device), reduction="sum")


def test_entropy_one_gradient_at_a_time(device):
    features, table, targets, _ = _problem(device, BF16, 500, 260, 96)
    both = torch.autograd.grad(vocabulary.linear_cross_entropy(features, table, targets), (features, table))
    only_f = torch.autograd.grad(vocabulary.linear_cross_entropy(features, table.detach(), targets), features)[0]
    only_t = torch.autograd.grad(vocabulary.linear_cross_entropy(features.detach(), table, targets), table)[0]
    assert torch.equal(both[0], only_f) and torch.equal(both[1], only_t)


def test_entropy_in_pieces(device):
    """More logits than one piece holds, in rows and in vocabulary, against the chunked definition on the GPU."""
    rows, vocab, dim = 70_001, 4_200, 8
    features, table, targets, _ = _problem(device, BF16, rows, vocab, dim, ignored=0.1)
    loss = vocabulary.linear_cross_entropy(features, table, targets)
    grads = torch.autograd.grad(loss, (features, table))
    count = int((targets != -100).sum())
    h, w = features.detach(), table.detach()
    total = bound = 0.0
    sums = [torch.zeros(vocab, dim, dtype=torch.float64, device=device) for _ in range(2)]
    for i in range(0, rows, 10_000):
        part = slice(i, i + 10_000)
        n = h[part].shape[0]
        want = ref.entropy(h[part], w, targets[part], torch.full((n,), 1.0 / count, device=device), reduction="none")
        total, bound = total + want["loss"][0].sum(), bound + want["loss"][1].sum()
        ref.check(grads[0][part], want["features"], "features")
        sums[0] += want["table"][0]
        sums[1] += want["table"][1]
    ref.check(loss, (total / count, bound / count + 2 * ref.U32 * total / count), "loss")
    ref.check(grads[1], (sums[0], sums[1] + sums[0].abs() * ref.ROUNDOFF[BF16] +
                         rows * ref.U32 * sums[0].abs()), "table")


def test_entropy_gradient_against_differences(device):
    """Central differences of the fp32 loss along random directions."""
    features, table, targets, gen = _problem(device, FP32, 37, 51, 20, spread=0.5)
    grads = torch.autograd.grad(vocabulary.linear_cross_entropy(features, table, targets, reduction="sum"),
                                (features, table))
    step = 2.0 ** -6
    for seed in range(4):
        d = [torch.randn(x.shape, generator=gen).to(device) for x in (features, table)]
        d = [x / x.norm() for x in d]

        def at(sign):
            with torch.no_grad():
                return vocabulary.linear_cross_entropy(features + sign * step * d[0], table + sign * step * d[1],
                                                       targets, reduction="none").double().sum().item()

        slope = (at(1.0) - at(-1.0)) / (2 * step)
        want = sum(float((g.double() * x.double()).sum()) for g, x in zip(grads, d))
        # losses to 37 rows' 2^-18 each over 2 steps; third derivatives of at most a few units in step^2 / 6
        assert abs(slope - want) <= 37 * 2.0 ** -18 / (2 * step) + 6.0 * step ** 2, (slope, want)


def test_tied_vocabulary_on_a_side_stream(device):
    """One table at both ends, on another stream than the default: the two gradients are added."""
    stream = torch.cuda.Stream()
    gen = _gen(5)
    tokens = torch.randint(0, 90, (400,), generator=gen).to(device)
    targets = torch.randint(0, 90, (400,), generator=gen).to(device)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        vocab = vocabulary.Vocabulary(90, 40, scale=2.0, padding_idx=0, logit_scale=0.5, device=device)
        features = vocab(tokens)
        features.retain_grad()
        loss = vocab.loss(features, targets)
        loss.backward()
    stream.synchronize()
    want = ref.entropy(features.detach(), vocab.weight.detach(), targets, 1.0, logit_scale=0.5)
    ref.check(loss, want["loss"], "loss")
    ref.check(features.grad, want["features"], "features")
    from_lookup = ref.embed_grad(tokens, features.grad, 90, 2.0, padding=0)
    ref.check(vocab.weight.grad, (want["table"][0] + from_lookup[0],
                                  want["table"][1] + from_lookup[1] + 4 * ref.U32 * (want["table"][0].abs() + from_lookup[0].abs())),
              "weight")


def test_vocabulary_operators_in_a_graph(device):
    """A training step captured once and replayed on new contents of its inputs."""
    gen = _gen(9)
    tokens = torch.randint(0, 300, (2000,), generator=gen).to(device)
    targets = torch.randint(0, 300, (2000,), generator=gen).to(device)
    targets[::9] = -100
    table = torch.randn(300, 64, generator=gen).to(device, BF16).requires_grad_(True)

    def step():
        features = vocabulary.embed_tokens(tokens, table, scale=1.5)
        loss = vocabulary.linear_cross_entropy(features, table, targets, logit_scale=0.3)
        return [loss.detach(), *torch.autograd.grad(loss, table)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        tokens.copy_(torch.randint(0, 300, (2000,), generator=_gen(seed)).to(device))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_refusals(device):
    table = torch.randn(10, 16, device=device)
    tokens = torch.zeros(4, dtype=torch.int64, device=device)
    features = torch.randn(4, 16, device=device)
    embed, entropy = vocabulary.embed_tokens, vocabulary.linear_cross_entropy
    for call, message in (
            (lambda: embed(tokens, table.double()), "dtype float32"),
            (lambda: embed(tokens, table[0]), "shape"),
            (lambda: embed(tokens, table[:0]), "shape"),
            (lambda: embed(tokens.float(), table), "int32 or int64"),
            (lambda: embed(tokens.cpu(), table), "must be on"),
            (lambda: embed([0], table), "torch.Tensor"),
            (lambda: embed(tokens, table, scale=math.nan), "finite"),
            (lambda: embed(tokens, table, padding_idx=10), "padding_idx"),
            (lambda: embed(tokens, table, padding_idx=-1), "padding_idx"),
            (lambda: entropy(features.half(), table, tokens), "dtype"),
            (lambda: entropy(features[:, :15], table, tokens), "shape"),
            (lambda: entropy(features, table, tokens[:3]), "targets must have shape"),
            (lambda: entropy(features, table, tokens.to(torch.uint8)), "int32 or int64"),
            (lambda: entropy(features, table, tokens, reduction="max"), "reduction"),
            (lambda: entropy(features, table, tokens, logit_scale=math.inf), "finite"),
            (lambda: entropy(features, table, tokens, ignore_index=1.5), "ignore_index"),
            (lambda: entropy(features.cpu(), table, tokens), "features must be")):
        with pytest.raises(ValueError, match=message):
            call()


@pytest.mark.parametrize("h_scale,w_scale,logit_scale", [(1e15, 1e-15, 1.0), (1e-20, 1.0, 1e20), (1e-20, 1e-20, 1.0),
                                                         (3e18, 3e18, 1e-36)])
def test_entropy_fp32_magnitudes(device, h_scale, w_scale, logit_scale):
    """fp32 features and tables far from 1, for short and for long rows."""
    for rows, vocab, dim in ((150, 90, 40), (150, 90, 200)):
        features, table, targets, gen = _problem(device, FP32, rows, vocab, dim)
        features = (features.detach() * h_scale).requires_grad_(True)
        table = (table.detach() * w_scale).requires_grad_(True)
        _compare(features, table, targets, torch.tensor(1.0, device=device), logit_scale=logit_scale)


@pytest.mark.parametrize("dim", [48, 144])
def test_entropy_fp32_rows_of_many_magnitudes(device, dim):
    """Rows and tables whose rows' sizes span six decades: as exact as fp32 for the largest of them."""
    features, table, targets, gen = _problem(device, FP32, 300, 200, dim)
    features = features.detach() * (10.0 ** (-6 * torch.rand(300, 1, generator=gen))).to(device)
    table = table.detach() * (10.0 ** (-6 * torch.rand(200, 1, generator=gen))).to(device)
    _compare(features.requires_grad_(True), table.requires_grad_(True), targets, torch.tensor(1.0, device=device),
             reduction="sum")


def test_language_scene_learns(device):
    from examples.language_scene import train

    losses = train(steps=12, count=4000, size=128)
    assert all(math.isfinite(x) for x in losses) and losses[-1] < 0.8 * losses[0]


def _marked(rows, dim, gen):
    """A few hundred row numbers: the ends, and both sides of the offsets that pass 2^31 and 2^32 bytes and elements."""
    at = [0, 1, rows - 1, rows - 2]
    for size in (2 ** 30, 2 ** 31, 2 ** 32):
        at += [r for r in (size // dim - 1, size // dim, size // dim + 1) if r < rows]
    return torch.cat([torch.tensor(at), torch.randint(0, rows, (300,), generator=gen)]).unique()


@pytest.mark.parametrize("dtype,rows,vocab,dim", [(BF16, 2 ** 24 + 5, 100, 136), (FP16, 2 ** 25 + 3, 70, 72),
                                                  (FP32, 2 ** 25 + 3, 50, 40), (FP32, 2 ** 23 + 1, 50, 260)])
def test_entropy_of_rows_past_32_bits(device, dtype, rows, vocab, dim):
    """The marked rows' losses, and gradients where only they have one; the others' terms are exact zeros."""
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim}", flush=True)
    gen = _gen(dim)
    marked = _marked(rows, dim, gen).to(device)
    features = torch.full((rows, dim), 0.25, dtype=dtype, device=device)
    features[marked] = torch.randn(len(marked), dim, generator=gen).to(device, dtype)
    table = (torch.randn(vocab, dim, generator=gen) / math.sqrt(dim)).to(device, dtype).requires_grad_(True)
    targets = torch.randint(0, vocab, (rows,), generator=gen, dtype=torch.int32).to(device)
    up = torch.zeros(rows, device=device)
    up[marked] = torch.rand(len(marked), generator=gen).to(device) + 0.5
    features.requires_grad_(True)
    loss = vocabulary.linear_cross_entropy(features, table, targets, reduction="none")
    want = ref.entropy(features.detach()[marked], table.detach(), targets[marked], up[marked], reduction="none")
    ref.check(loss.detach()[marked], want["loss"], "loss")
    grad_features, grad_table = torch.autograd.grad(loss, (features, table), up)
    ref.check(grad_features[marked], want["features"], "features")
    ref.check(grad_table, want["table"], "table")
    grad_features[marked] = 0
    assert not grad_features.any()


@pytest.mark.parametrize("dtype,rows,vocab,dim", [(BF16, 33, 2 ** 24 + 5, 136), (FP16, 300, 2 ** 25 + 1, 72),
                                                  (FP32, 70, 2 ** 23 + 1, 136), (BF16, 300, 2 ** 23 + 1, 264)])
def test_entropy_of_tables_past_32_bits(device, dtype, rows, vocab, dim):
    """Marked rows of the table hold all but 2^-30 of every probability; the others are zeros, of logit 0."""
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim}", flush=True)
    gen = _gen(dim)
    marked = _marked(vocab, dim, gen).to(device)
    table = torch.zeros(vocab, dim, dtype=dtype, device=device)
    table[marked] = (torch.randn(len(marked), dim, generator=gen) / math.sqrt(dim)).to(device, dtype)
    features = (30.0 * torch.sign(torch.randn(rows, dim, generator=gen))).to(device, dtype).requires_grad_(True)
    label = torch.randint(0, len(marked), (rows,), generator=gen).to(device)
    few = table[marked]
    lse = torch.logsumexp(features.detach().double() @ few.double().T, 1)
    rest = vocab * torch.exp(-lse)
    assert float(rest.max()) < 2.0 ** -30
    up = torch.rand(rows, generator=gen).to(device) + 0.5
    want = ref.entropy(features.detach(), few, label, up, reduction="none")
    table.requires_grad_(True)
    loss = vocabulary.linear_cross_entropy(features, table, marked[label], reduction="none")
    ref.check(loss, want["loss"], "loss")
    grad_features, grad_table = torch.autograd.grad(loss, (features, table), up)
    ref.check(grad_features, want["features"], "features")
    value, bound = want["table"]
    if dtype == FP32:
        # the gradients of the logits are held as three planes of 22 bits in steps of 2^-62 of the largest
        bound = bound + 2.0 ** -62 * up.max().double() * features.detach().double().abs().sum(0)
    ref.check(grad_table[marked], (value, bound), "table")
    grad_table[marked] = 0
    assert float(grad_table.abs().max()) <= rows * 30.0 * 1.5 * 2.0 ** -30


def test_lookup_of_more_vectors_than_a_launch_has_threads(device):
    n, dim = 2 ** 30 + 77, 16  # two vectors a row
    table = torch.randn(5, dim, generator=_gen(4)).to(device, BF16)
    tokens = torch.arange(n, dtype=torch.int32, device=device) % 5
    out = vocabulary.embed_tokens(tokens, table)
    for at in (0, 2 ** 27, 2 ** 28, 2 ** 29, 2 ** 30 - 100, n - 100):
        assert torch.equal(out[at:at + 100], table[tokens[at:at + 100]])


@pytest.mark.parametrize("dtype,rows,vocab,dim", [
    (FP32, 70_001, 1000, 40), (FP32, 70_001, 1000, 136), (FP16, 130_003, 520, 100), (BF16, 130_003, 520, 9),
    (FP32, 1_100_003, 64, 8), (FP32, 1_100_003, 64, 72), (BF16, 66_001, 8192, 72), (FP16, 66_001, 8192, 136)])
@pytest.mark.parametrize("ignored", [0.0, 0.4, "half", "all but one"])
def test_entropy_of_many_rows_of_which_some_count(device, dtype, rows, vocab, dim, ignored):
    """Sizes at which the rows that count are put first: with and without a gradient, in one piece and in several."""
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim} ignored={ignored}", flush=True)
    gen = torch.Generator(device=device).manual_seed(dim)
    features = torch.randn(rows, dim, generator=gen, device=device).to(dtype)
    table = (torch.randn(vocab, dim, generator=gen, device=device) / math.sqrt(dim)).to(dtype).requires_grad_(True)
    targets = torch.randint(0, vocab, (rows,), generator=gen, device=device)
    if ignored == "half":
        out = torch.arange(rows, device=device) < rows // 2
    elif ignored == "all but one":
        out = torch.arange(rows, device=device) != rows - 3
    else:
        out = torch.rand(rows, generator=gen, device=device) < ignored
    targets[out] = -100
    features[out] = math.nan
    features.requires_grad_(True)
    up = torch.rand(rows, generator=gen, device=device) + 0.5
    loss = vocabulary.linear_cross_entropy(features, table, targets, reduction="none")
    grads = torch.autograd.grad(loss, (features, table), up)
    with torch.no_grad():
        assert torch.equal(loss, vocabulary.linear_cross_entropy(features, table, targets, reduction="none"))
        mean = vocabulary.linear_cross_entropy(features, table, targets)
    assert not loss[out].any() and not grads[0][out].any()
    # the rows that count, a part of them at a time; the table's gradient from the bounds of all parts
    kept = (~out).nonzero().squeeze(1)
    total, value, bound = 0.0, 0.0, 0.0
    for ids in kept.split(max(1, 2 ** 26 // vocab)):
        want = ref.entropy(features.detach()[ids], table.detach(), targets[ids], up[ids], reduction="none")
        ref.check(loss[ids], want["loss"], "loss")
        ref.check(grads[0][ids], want["features"], "features")
        total += float(want["loss"][0].sum())
        value, bound = value + want["table"][0], bound + want["table"][1]
    ref.check(grads[1], (value, bound), "table")
    assert abs(float(mean) - total / len(kept)) <= 1e-5 * max(1.0, abs(total / len(kept)))


@pytest.mark.parametrize("dim", [1, 8, 13])
def test_lookup_of_short_rows_is_few_launches(device, dim):
    """Rows of one vector: a pass costs what its bytes do, not a launch for each row."""
    table = torch.randn(34, dim, generator=_gen(dim)).to(device, BF16)
    tokens = torch.randint(0, 34, (300_001,), generator=_gen(dim)).to(device)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as trace:
        out = vocabulary.embed_tokens(tokens, table)
        torch.cuda.synchronize()
    assert torch.equal(out, table[tokens])
    assert sum(e.count for e in trace.key_averages() if "lookup" in e.key) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,dim,rows", [(5, 367, 40_000), (5, 64, 40_000), (129, 264, 20_000), (70, 200, 9)])
def test_entropy_mean_of_small_losses_has_no_bias(device, dtype, vocab, dim, rows):
    """Labels that lead by about 8: the rows' errors are roundings and average out.

    A loss below 1/8 is the logarithm of 1 and a sum that fp32 rounds to 2^-24 once or twice, and of
    terms whose exponents (up to 16 in base 2) are rounded to 2^-20: 2^-23 in all for a row, with
    either sign, so 8 standard errors of the mean are 2^-20 / sqrt(rows), besides the fp32 scale's own 2^-25 of 8 times a loss.
    """
    gen = _gen(dim)
    table = torch.randn(vocab, dim, generator=gen, dtype=torch.float64) / math.sqrt(dim)
    label = torch.randint(0, vocab, (rows,), generator=gen)
    features = torch.randn(rows, dim, generator=gen, dtype=torch.float64) + 8.0 * table[label]
    features, table, label = features.to(device, dtype), table.to(device, dtype), label.to(device)
    s = features.double() @ table.double().T
    loss = torch.logsumexp(s, 1) - s.gather(1, label.unsqueeze(1)).squeeze(1)
    got = vocabulary.linear_cross_entropy(features, table, label, reduction="none").double()
    small = loss < 0.125
    assert int(small.sum()) > rows // 4
    bias = float((got - loss)[small].mean())
    assert abs(bias) <= 2.0 ** -20 / math.sqrt(int(small.sum())) + 2.0 ** -22 * float(loss[small].mean()), bias


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,dim", [(257, 320), (129, 320), (65, 64), (65, 320), (1025, 128)])
def test_entropy_of_a_table_row_of_nan(device, dtype, vocab, dim):
    """The last row of the table alone in its tile: no row's loss is a number."""
    features, table, targets, gen = _problem(device, dtype, 700, vocab, dim, ignored=0.0)
    table = table.detach().clone()
    table[-1] = math.nan
    assert torch.isnan(vocabulary.linear_cross_entropy(features.detach(), table, targets, reduction="none")).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocab,dim", [(70_000, 1, 24), (40_000, 2, 16), (30_000, 3, 128), (40, 1700, 64),
                                            (1, 66_000, 40), (5001, 67, 100), (1030, 65, 7), (300, 257, 72),
                                            (2, 40_000, 128), (9000, 128, 1)])
def test_entropy_of_short_rows_in_one_plane(device, dtype, rows, vocab, dim):
    """16-bit rows of up to 128 values with logits enough for the kernels that keep them in registers."""
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim}", flush=True)
    features, table, targets, gen = _problem(device, dtype, rows, vocab, dim, ignored=0.2 if rows > 2 else 0.0)
    features = features.detach().clone()
    features[targets == -100] = math.nan
    features.requires_grad_(True)
    for reduction, logit_scale in (("mean", 1.0), ("none", -1.5), ("sum", 0.0)):
        up = torch.rand(rows, generator=gen).to(device) if reduction == "none" else torch.tensor(0.5, device=device)
        _compare(features, table, targets, up, reduction=reduction, logit_scale=logit_scale)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,vocab,dim", [(5, 42, 640), (1, 2, 1), (38, 8192, 768), (700, 90, 128), (200, 2000, 300)])
def test_entropy_of_few_rows_rounds_once(device, dtype, rows, vocab, dim):
    """The gradients' distance from 64 bits is that of their own rounding and a tenth of it."""
    print(f"entropy {dtype} rows={rows} vocab={vocab} dim={dim}", flush=True)
    features, table, targets, gen = _problem(device, dtype, rows, vocab, dim, ignored=0.0)
    want = ref.entropy(features.detach(), table.detach(), targets, 8.0, reduction="sum")
    loss = vocabulary.linear_cross_entropy(features, table, targets, reduction="sum")
    grads = torch.autograd.grad(loss, (features, table), torch.tensor(8.0, device=device))
    for name, got in zip(("features", "table"), grads):
        value = want[name][0]
        own = (value.to(dtype).double() - value).norm()
        assert float((got.double() - value).norm()) <= 1.1 * float(own) + 1e-6 * float(value.norm()), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 2, 4, 7, 12, 33, 64, 130, 300])
@pytest.mark.parametrize("lengths", [
    [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17] * 40, [63, 64, 65, 127, 128, 129, 255, 256, 257] * 4,
    [511, 512, 513, 1, 1023, 1024, 1025, 1, 2047, 2048, 2049], [1, 30_000, 1], [4096] * 5])
def test_lookup_gradient_runs_of_every_length(device, dtype, dim, lengths):
    """Runs that begin and end at parts, waves and chunks, for rows of one lane to rows of many: of whole
    numbers, so that every order of the sums gives the same."""
    gen = _gen(dim + len(lengths))
    vocab = 2 * len(lengths) + 1  # every other row is named by no token
    tokens = torch.repeat_interleave(2 * torch.arange(len(lengths)) + 1, torch.tensor(lengths))
    tokens = tokens[torch.randperm(tokens.numel(), generator=gen)]
    up = torch.randint(-4, 5, (tokens.numel(), dim), generator=gen).float()
    expected = torch.zeros(vocab, dim).index_add_(0, tokens, up).to(dtype)
    table = torch.zeros(vocab, dim, dtype=dtype, device=device, requires_grad=True)
    (grad,) = torch.autograd.grad(vocabulary.embed_tokens(tokens.to(device), table), table, up.to(device, dtype))
    assert torch.equal(grad.cpu(), expected)
