"""The vocabulary operators' checks that need no GPU: the Python refusals, the C ABI's statuses and
workspace sizes."""

from __future__ import annotations

import pytest
import torch

import gswarp.vocabulary as alias
from gswarp_amd import _lib, vocabulary
import vocabulary_ref as ref


def test_alias_and_host_tensors():
    assert alias.embed_tokens is vocabulary.embed_tokens and alias.Vocabulary is vocabulary.Vocabulary
    with pytest.raises(ValueError, match="CUDA tensor"):
        vocabulary.embed_tokens(torch.zeros(1, dtype=torch.int64), torch.zeros(2, 2))
    with pytest.raises(ValueError, match="CUDA tensor"):
        vocabulary.linear_cross_entropy(torch.zeros(1, 2), torch.zeros(2, 2), torch.zeros(1, dtype=torch.int64))


def test_vocabulary_module_initialises():
    v = vocabulary.Vocabulary(7, 5, scale=2.0, padding_idx=1, dtype=torch.bfloat16)
    assert v.weight.shape == (7, 5) and v.weight.dtype == torch.bfloat16 and v.weight.requires_grad


@pytest.fixture
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libgswarp_hip.so not built")
    return _lib.load()


def test_statuses_before_any_launch(lib):
    p = 4096  # an aligned address that no refused call reads
    ok = dict(n=4, vocab=10, dim=16, dtype=1, tokens=p, bits=64, table=p, ld=16, scale=1.0, out=p)

    def embed(**kw):
        return lib.gs_embed_fwd(*{**ok, **kw}.values(), None)

    for bad in (dict(n=-1), dict(vocab=0), dict(dim=0), dict(dtype=3), dict(dtype=-1), dict(bits=16), dict(tokens=None),
                dict(table=None), dict(out=None), dict(ld=15), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert embed(**bad) == -1, bad
    assert embed(n=2 ** 31) == -4 and embed(dim=2 ** 22, ld=2 ** 22) == -4
    assert embed(n=0) == 0
    assert lib.gs_embed_bwd(4, 10, 16, 1, p, 64, p, 1.0, -1, p, p, 16, None) == -3
    assert lib.gs_embed_bwd(4, 10, 16, 1, p, 64, p, 1.0, -1, p, p + 8, 1 << 30, None) == -2
    assert lib.gs_embed_bwd(4, 10, 16, 1, p, 64, None, 1.0, -1, p, p, 1 << 30, None) == -1

    fwd = dict(rows=4, vocab=10, dim=16, dtype=1, features=p, ldf=16, table=p, ldt=16, targets=p, bits=64, ignore=-100,
               scale=1.0, reduction=2, loss=p, lse=p, count=p, workspace=p, nbytes=1 << 40)

    def entropy(**kw):
        return lib.gs_xent_fwd(*{**fwd, **kw}.values(), None)

    for bad in (dict(rows=-1), dict(vocab=0), dict(dim=0), dict(dtype=7), dict(features=None), dict(table=None),
                dict(targets=None), dict(bits=8), dict(scale=float("inf")), dict(reduction=3), dict(loss=None),
                dict(count=None), dict(ldf=8), dict(ldt=15)):
        assert entropy(**bad) == -1, bad
    assert entropy(nbytes=64) == -3 and entropy(workspace=None) == -3
    assert entropy(features=p + 2) == -2 and entropy(table=p + 8) == -2 and entropy(workspace=p + 16) == -2
    assert entropy(rows=2 ** 31) == -4
    bwd = dict(rows=4, vocab=10, dim=16, dtype=1, features=p, ldf=16, table=p, ldt=16, targets=p, bits=64, ignore=-100,
               scale=1.0, reduction=2, lse=p, count=p, grad=p, gf=p, gt=p, workspace=p, nbytes=1 << 40)

    def entropy_bwd(**kw):
        return lib.gs_xent_bwd(*{**bwd, **kw}.values(), None)

    for bad in (dict(lse=None), dict(count=None), dict(grad=None), dict(reduction=-1), dict(targets=None)):
        assert entropy_bwd(**bad) == -1, bad
    assert entropy_bwd(nbytes=64) == -3
    assert entropy_bwd(gf=None, gt=None) == 0  # nothing asked, nothing launched


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspaces_do_not_grow_with_the_logits(lib, dtype):
    """Rows x vocabulary of a million by a hundred thousand would be 200 GB in 16 bits."""
    rows, vocab, dim = 1_000_000, 100_000, 64
    inputs = (rows + vocab) * dim * 6
    assert lib.gs_xent_fwd_workspace_bytes(rows, vocab, dim, dtype, dim, dim) < (1 << 30) + inputs
    assert lib.gs_xent_bwd_workspace_bytes(rows, vocab, dim, dtype, dim, dim, 1, 1) < 2 * (1 << 30) + 4 * inputs
    assert lib.gs_xent_fwd_workspace_bytes(0, vocab, dim, dtype, dim, dim) == 0
    assert lib.gs_embed_bwd_workspace_bytes(0, vocab, dim, dtype) == 0
    assert lib.gs_embed_bwd_workspace_bytes(rows, vocab, dim, dtype) > 16 * rows


def test_reference_agrees_with_autograd():
    """The 64-bit reference used by the GPU tests against torch's own cross entropy."""
    gen = torch.Generator().manual_seed(0)
    h = torch.randn(30, 8, generator=gen, dtype=torch.float64).requires_grad_(True)
    w = torch.randn(11, 8, generator=gen, dtype=torch.float64).requires_grad_(True)
    t = torch.randint(0, 11, (30,), generator=gen)
    t[::4] = -100
    for reduction in ("mean", "sum", "none"):
        up = torch.rand(30, generator=gen, dtype=torch.float64) if reduction == "none" else torch.tensor(0.3, dtype=torch.float64)
        loss = torch.nn.functional.cross_entropy(0.7 * h @ w.T, t, reduction=reduction)
        grads = torch.autograd.grad(loss, (h, w), up)
        f32 = ref.entropy(h.detach().float(), w.detach().float(), t, up, reduction=reduction, logit_scale=0.7)
        assert torch.allclose(loss, f32["loss"][0], atol=1e-5)
        assert torch.allclose(grads[0], f32["features"][0], atol=1e-5)
        assert torch.allclose(grads[1], f32["table"][0], atol=1e-5)


def test_limits_and_alignment_of_gradients(lib):
    p = 4096
    sizes = (4, 10, 16, 1, p, 16, p, 16, p, 64, -100, 1.0, 2)
    assert lib.gs_xent_bwd(*sizes, p, p, p, p + 8, p, p, 1 << 40, None) == -2
    assert lib.gs_xent_bwd(*sizes, p, p, p, p, p + 4, p, 1 << 40, None) == -2
    wide = (4, 2 ** 29 + 1, 16, 1, p, 16, p, 16, p, 64, -100, 1.0, 2)
    assert lib.gs_xent_fwd(*wide, p, p, p, p, 1 << 40, None) == -4
