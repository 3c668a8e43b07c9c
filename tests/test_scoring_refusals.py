"""What the token score and distillation calls refuse, checked on the CPU.

Every refusal comes before anything touches a device, so the addresses here
are never read; a call that passes its checks ends at the missing device.
"""
import numpy as np
import pytest

OK, EMPTY, TOO_MANY, INVALID, NO_DEVICE = 0, 32, 36, 63, 65
P = 1 << 20  # an aligned address that is never read
F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    import detllm_b200 as D

    if D.device_count() > 0:
        pytest.skip("a GPU is visible: an accepted call would run")
    return D.lib()


def scores(lib, x=P, dtype=F32, n=4, vocab=1000, ld=1000, tok=P, tb=8, top=0, lp=P, en=P, st=P, ids=None, lps=None, ws=P, size=1 << 40):
    return lib.det_token_scores_device(x, dtype, n, vocab, ld, tok, tb, top, lp, en, st, ids, lps, None, ws, size, None)


def scores_grad(lib, x=P, dtype=F32, n=4, vocab=1000, ld=1000, tok=P, tb=8, st=P, gl=P, ge=None, out=P, old=1000):
    return lib.det_token_scores_grad_device(x, dtype, n, vocab, ld, tok, tb, st, gl, ge, out, old, None)


def scores_step(lib, x=P, dtype=F32, n=4, vocab=1000, ld=1000, tok=P, tb=8, gl=P, ge=None, lp=P, en=P, st=P, out=P,
                old=1000, ws=P, size=1 << 40):
    return lib.det_token_scores_step_device(x, dtype, n, vocab, ld, tok, tb, gl, ge, lp, en, st, out, old, None, ws,
                                            size, None)


def loss(lib, x=P, dtype=F32, n=4, vocab=1000, ld=1000, ids=P, ib=4, u=P, ud=F32, k=8, lld=8, t=1.0, out=P, st=P,
         ws=P, size=1 << 40):
    return lib.det_distill_loss_device(x, dtype, n, vocab, ld, ids, ib, u, ud, k, lld, t, out, st, None, ws, size,
                                       None)


def loss_grad(lib, x=P, dtype=F32, n=4, vocab=1000, ld=1000, ids=P, ib=4, u=P, ud=F32, k=8, lld=8, t=1.0, st=P, g=P,
              out=P, old=1000):
    return lib.det_distill_grad_device(x, dtype, n, vocab, ld, ids, ib, u, ud, k, lld, t, st, g, out, old, None)


def loss_step(lib, x=P, dtype=F32, n=4, vocab=1000, ld=1000, ids=P, ib=4, u=P, ud=F32, k=8, lld=8, t=1.0, g=P, lo=P,
              st=P, out=P, old=1000, ws=P, size=1 << 40):
    return lib.det_distill_step_device(x, dtype, n, vocab, ld, ids, ib, u, ud, k, lld, t, g, lo, st, out, old, None,
                                       ws, size, None)


ALL = [scores, scores_grad, scores_step, loss, loss_grad, loss_step]
GRADS = [scores_grad, scores_step, loss_grad, loss_step]
LISTS = [loss, loss_grad, loss_step]


@pytest.mark.parametrize("call", ALL)
def test_logits(lib, call):
    assert call(lib) == NO_DEVICE  # the call itself is fine
    assert call(lib, n=0, x=None) == OK
    assert call(lib, x=None) == INVALID
    assert call(lib, dtype=3) == INVALID
    assert call(lib, dtype=-1) == INVALID
    assert call(lib, vocab=0) == EMPTY
    assert call(lib, vocab=(1 << 18) + 1) == TOO_MANY
    assert call(lib, n=(1 << 26) + 1) == INVALID
    assert call(lib, x=P + 2) == INVALID  # f32 rows at a 2-byte address
    assert call(lib, x=P + 1, dtype=BF16) == INVALID
    assert call(lib, ld=1 << 41) == INVALID


def test_rows_that_overlap_may_be_read(lib):
    assert scores(lib, ld=0) == NO_DEVICE  # one row, n times
    assert loss(lib, ld=7) == NO_DEVICE


@pytest.mark.parametrize("call", [scores, scores_grad, scores_step])
def test_tokens(lib, call):
    assert call(lib, tok=None) == INVALID
    assert call(lib, tb=2) == INVALID
    assert call(lib, tok=P + 4) == INVALID
    assert call(lib, tok=P + 4, tb=4) == NO_DEVICE


def test_tokens_that_nothing_needs(lib):
    assert scores(lib, tok=None, lp=None) == NO_DEVICE
    assert scores_grad(lib, tok=None, gl=None, ge=P) == NO_DEVICE
    assert scores_step(lib, tok=None, gl=None, ge=P, lp=None) == NO_DEVICE


def test_top(lib):
    assert scores(lib, top=5) == INVALID  # nowhere to put it
    assert scores(lib, top=5, ids=P) == NO_DEVICE
    assert scores(lib, top=128, ids=P, lps=P) == NO_DEVICE
    assert scores(lib, top=129, ids=P, lps=P) == INVALID
    assert scores(lib, top=6, vocab=5, ids=P, lps=P) == INVALID


@pytest.mark.parametrize("call", [scores, loss])
def test_workspace(lib, call):
    need = lib.det_scores_workspace(F32, 4, 1000, 0)
    assert need > 0
    assert call(lib, size=need) == NO_DEVICE
    assert call(lib, size=need - 1) == INVALID
    assert call(lib, ws=None) == INVALID
    assert call(lib, ws=P + 8) == INVALID
    assert lib.det_scores_workspace(F32, 4, 1000, 5) > need  # a top list keeps more
    assert lib.det_scores_workspace(F32, 4, (1 << 18) + 1, 0) == 0
    assert lib.det_scores_workspace(3, 4, 1000, 0) == 0


@pytest.mark.parametrize("call,k", [(scores_step, 1), (loss_step, 8)])
def test_step_workspace(lib, call, k):
    need = lib.det_step_workspace(4, 1000, k)
    assert need > 0
    assert call(lib, size=need) == NO_DEVICE
    assert call(lib, size=need - 1) == INVALID
    assert call(lib, ws=None) == INVALID
    assert call(lib, ws=P + 8) == INVALID
    assert lib.det_step_workspace(4, 1000, 129) == 0


@pytest.mark.parametrize("call", LISTS)
def test_lists(lib, call):
    assert call(lib, ids=None) == INVALID
    assert call(lib, u=None) == INVALID
    assert call(lib, ud=5) == INVALID
    assert call(lib, u=P + 2) == INVALID
    assert call(lib, u=P + 2, ud=F16) == NO_DEVICE
    assert call(lib, ib=1) == INVALID
    assert call(lib, ids=P + 4, ib=8) == INVALID
    assert call(lib, k=0) == INVALID
    assert call(lib, k=129, lld=129) == INVALID
    assert call(lib, k=9) == INVALID  # lists of 9 every 8 entries
    for t in (0.0, -1.0, 1e-7, 1e7, float("inf"), float("nan")):
        assert call(lib, t=t) == INVALID, t
    assert call(lib, t=1e-6) == NO_DEVICE
    assert call(lib, t=1e6) == NO_DEVICE


@pytest.mark.parametrize("call", GRADS)
def test_gradient_places(lib, call):
    size = 4 * 4000
    assert call(lib, out=None) == INVALID
    assert call(lib, old=999) == INVALID  # rows of the gradient overlap
    assert call(lib, out=P + 2) == INVALID
    assert call(lib, out=P + size) == NO_DEVICE  # behind the logits
    assert call(lib, out=P - size) == NO_DEVICE  # before them
    assert call(lib, out=P + 4) == INVALID  # over them, shifted
    assert call(lib, out=P + size - 4) == INVALID
    assert call(lib, out=P - size + 4) == INVALID
    assert call(lib, ld=2000) == INVALID  # over them, with another stride
    assert call(lib, ld=2000, old=2000) == NO_DEVICE
    assert call(lib, ld=2000, old=2000, out=P + 4000) == NO_DEVICE  # side by side
    assert call(lib, ld=2000, old=2000, out=P - 4000) == NO_DEVICE
    assert call(lib, ld=2000, old=2000, out=P + 4004) == INVALID  # into the next row
    assert call(lib, ld=2000, old=2000, out=P + 3996) == INVALID
    assert call(lib, ld=2000, old=2000, out=P - 3996) == INVALID
    assert call(lib, ld=0) == INVALID  # one row of logits, n of gradients over it


def test_what_a_gradient_needs(lib):
    assert scores_grad(lib, st=None) == INVALID
    assert scores_grad(lib, gl=None) == INVALID
    assert scores_step(lib, st=None) == INVALID
    assert scores_step(lib, gl=None) == INVALID
    assert loss(lib, out=None) == INVALID
    assert loss_grad(lib, st=None) == INVALID
    assert loss_grad(lib, g=None) == INVALID
    assert loss_step(lib, g=None) == INVALID
    assert loss_step(lib, lo=None) == INVALID
    assert loss_step(lib, st=None) == INVALID


def test_session_calls_without_a_session(lib):
    assert lib.det_token_scores(None, None, P, 1, 0, P, P, None, None) == INVALID
    assert lib.det_distill_loss(None, None, 1, P, P, 1, 1.0, P) == INVALID


def test_tensors_that_are_not_on_a_device():
    import torch

    from detllm_b200 import scoring

    x, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    one = torch.ones(3)
    lists = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    for call in (lambda: scoring.token_scores(x, t), lambda: scoring.token_scores_grad(x, t, torch.zeros(3, 4), one),
                 lambda: scoring.token_scores_step(x, t, one), lambda: scoring.distill_loss(x, *lists),
                 lambda: scoring.distill_grad(x, *lists, torch.zeros(3, 4), one),
                 lambda: scoring.distill_step(x, *lists, one)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def windows(n, n_ctx):
    """(window start, tokens read there) of Model.score's loop, for a model
    whose session only records what it is asked."""
    import detllm_b200 as D

    seen = {}

    class Config:
        context_length = 1 << 20

    class Fake:
        config, vocab, calls = Config, 50, []
        score = D.Model.score

    class Session:
        def __init__(self, model, n_ctx, chunk):
            self.n_ctx, self.max_chunk, self.kv = n_ctx, min(chunk, 3), []

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            pass

        def reset(self):
            self.kv = []

        def forward(self, t, pos0):
            assert pos0 == len(self.kv) and pos0 + len(t) <= self.n_ctx
            self.kv += list(t)
            self.first = pos0

        def token_scores(self, tokens, rows, top):
            for j, tok in zip(rows, tokens):
                seen[int(tok)] = self.kv[: self.first + int(j) + 1]
            z = np.zeros(len(tokens), np.float32)
            return z, z, np.zeros((len(tokens), top)), np.zeros((len(tokens), top))

    old = D.Session
    D.Session = Session
    try:
        lp, _, ids, _ = Fake().score(np.arange(n), n_ctx, 2)
    finally:
        D.Session = old
    return lp, seen, ids


@pytest.mark.parametrize("n,n_ctx", [(1, 8), (2, 8), (8, 8), (9, 8), (30, 8), (31, 12), (20, 3), (7, 2), (5, 1)])
def test_score_reads_each_token_in_the_codec_s_context(n, n_ctx):
    lp, seen, ids = windows(n, n_ctx)
    # det-cli's state machine, one token at a time (main.rs:632-778)
    start, overlap = 0, n_ctx // 4
    for pos in range(n):
        if pos - start >= n_ctx:
            start = pos - overlap
        context = list(range(start, pos))
        if context:
            assert seen[pos] == context
        else:
            assert pos not in seen and lp[pos] == np.float32(-np.log(50)) and list(ids[pos]) == [0, 1]
