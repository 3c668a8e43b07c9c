"""Rows of which several things are wrong at once, as include/detgpu.h orders
them, on each of the kernels that may take the call."""
import pytest

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
SHAPES = [(500, "float32"), (30000, "float16"), (50000, "bfloat16")]


def same(torch, got, want):
    want = torch.tensor(want, device="cuda")
    return torch.equal(torch.nan_to_num(got, nan=77.0, posinf=88.0, neginf=99.0),
                       torch.nan_to_num(want, nan=77.0, posinf=88.0, neginf=99.0))


@pytest.mark.parametrize("vocab,dtype", SHAPES)
def test_tokens(vocab, dtype):
    import torch

    from detllm_b200 import scoring as sc

    x = torch.randn(6, vocab, device="cuda").to(getattr(torch, dtype))
    x[[0, 1, 2]] = -INF  # nothing is left
    x[[3, 4], 9] = NAN
    tokens = torch.tensor([-1, vocab, 3, -1, vocab, -1], device="cuda")
    lp = [0.0, NAN, -INF, NAN, NAN, 0.0]
    one = torch.ones(6, device="cuda")
    for top in (0, 5):
        f = sc.token_scores(x, tokens, top=top)
        assert same(torch, f.logprob, lp)
        assert same(torch, f.entropy[:5], [0.0, 0.0, 0.0, NAN, NAN])
        if top:
            assert f.top_ids[:3].tolist() == [[0, 1, 2, 3, 4]] * 3 and (f.top_ids[3:5] == -1).all()
    for gl, gh in ((one, None), (one, one), (None, one)):
        r, step = sc.token_scores_step(x, tokens, gl, gh)
        assert same(torch, r.logprob, lp)
        for grad in (step, sc.token_scores_grad(x, tokens, f.stats, gl, gh)):
            assert (grad[:3] == 0).all() and torch.isnan(grad[3:5]).all()
            assert torch.isfinite(grad[5]).all() and bool((grad[5] != 0).any()) == (gh is not None)


@pytest.mark.parametrize("vocab,dtype", SHAPES)
def test_lists(vocab, dtype):
    import torch

    from detllm_b200 import scoring as sc

    x = torch.randn(7, vocab, device="cuda").to(getattr(torch, dtype))
    x[[0, 1, 2]] = -INF
    x[[3, 4, 5], 9] = INF
    ids = torch.arange(4, device="cuda").repeat(7, 1)
    u = torch.randn(7, 4, device="cuda")
    ids[0], ids[1, 2], ids[3], ids[4, 2] = -1, vocab, -1, vocab
    u[6, :2] = -INF  # not valid; the rest is
    want = [0.0, NAN, INF, 0.0, NAN, NAN]
    one = torch.ones(7, device="cuda")
    f = sc.distill_loss(x, ids, u, 2.0)
    r, step = sc.distill_step(x, ids, u, one, 2.0)
    assert same(torch, f.loss[:6], want) and same(torch, r.loss[:6], want)
    assert torch.isfinite(f.loss[6]) and torch.equal(f.loss[6], r.loss[6])
    for grad in (step, sc.distill_grad(x, ids, u, f.stats, one, 2.0)):
        assert (grad[:4] == 0).all() and torch.isnan(grad[4:6]).all() and torch.isfinite(grad[6]).all()
