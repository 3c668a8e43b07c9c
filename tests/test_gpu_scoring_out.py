"""The gradient's ``out``, where autograd knows the tensor."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def calls():
    import torch

    from detllm_b200 import scoring as sc

    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(5, 3001, generator=g, device="cuda")
    tokens = torch.randint(0, 3001, (5,), generator=g, device="cuda")
    one = torch.ones(5, device="cuda")
    f = sc.token_scores(x.exp(), tokens, top=9)
    ids, u = f.top_ids, f.top_logprobs
    return torch, x, {
        "scores grad": lambda y, o: sc.token_scores_grad(y, tokens, f.stats, one, out=o),
        "scores step": lambda y, o: sc.token_scores_step(y, tokens, one, out=o)[1],
        "distill grad": lambda y, o: sc.distill_grad(y, ids, u, f.stats, one, out=o),
        "distill step": lambda y, o: sc.distill_step(y, ids, u, one, out=o)[1],
    }


OPS = ["scores grad", "scores step", "distill grad", "distill step"]


@pytest.mark.parametrize("op", OPS)
def test_logits_that_a_backward_needs(calls, op):
    """exp's backward needs its result: with the gradient written over it, it is
    refused, as after any change in place."""
    torch, x, ops = calls
    leaf = x.clone().requires_grad_()
    logits = leaf.exp()
    want = ops[op](logits, None)
    assert logits._version == 0
    got = ops[op](logits.detach(), logits.detach())
    assert torch.equal(got, want) and torch.equal(logits, want)
    with pytest.raises(RuntimeError, match="inplace"):
        logits.sum().backward()


@pytest.mark.parametrize("op", OPS)
def test_logits_that_no_backward_needs(calls, op):
    """A product's backward does not need its result: the gradient may be
    written over it and handed on."""
    torch, x, ops = calls
    leaf = x.exp().requires_grad_()
    logits = 1.0 * leaf
    grad = ops[op](logits.detach(), logits.detach())
    logits.backward(grad)
    assert torch.equal(leaf.grad, ops[op](leaf.detach(), None))


@pytest.mark.parametrize("op", OPS)
def test_tensors_without_a_version(calls, op):
    torch, x, ops = calls
    want = ops[op](x.exp(), None)
    with torch.inference_mode():
        y = x.exp()
        assert torch.equal(ops[op](y, y), want)
