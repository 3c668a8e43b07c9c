"""Calls right behind one another on the same tensors: each kernel may start
before its predecessor ends, and reads what that left all the same."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,vocab", [(5, 1500), (40, 30000), (3, 50001), (700, 9001)])
def test_scores_of_what_the_call_before_wrote(n, vocab, dtype):
    """Gradients written over the logits, scored, and so on, in a stream and in
    a graph, against the same calls with a wait between them."""
    import torch

    from detllm_b200 import scoring as sc

    g = torch.Generator(device="cuda").manual_seed(n)
    start = (torch.randn(n, vocab, generator=g, device="cuda") * 3).to(getattr(torch, dtype))
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    one = torch.full((n,), 50.0, device="cuda")
    ids = torch.randint(0, vocab, (n, 7), generator=g, device="cuda")
    u = torch.randn(n, 7, generator=g, device="cuda")

    def chain(x, between):
        seen = []

        def keep(*tensors):
            seen.extend(tensors)
            between()

        for top in (0, 3):
            f = sc.token_scores(x, tokens, top=top)
            keep(*f[:3])
            sc.token_scores_grad(x, tokens, f.stats, one, one, out=x)
            between()
            f = sc.token_scores(x, tokens, top=top)
            keep(*f[: 5 if top else 3])
            keep(*sc.distill_step(x, ids, u, one, 0.5, out=x)[0])
            keep(*sc.distill_loss(x, ids, u, 0.5))
            keep(*sc.token_scores_step(x, tokens, one, one, out=x)[0][:3])
            keep(*sc.token_scores(x, tokens, top=top)[: 5 if top else 3])
        seen.append(x.clone())
        return seen

    want = chain(start.clone(), torch.cuda.synchronize)
    x = torch.empty_like(start)
    for _ in range(20):
        x.copy_(start)
        got = chain(x, lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x.copy_(start)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = chain(x, lambda: None)
    for _ in range(20):
        x.copy_(start)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
