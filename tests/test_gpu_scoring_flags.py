"""What a call reports of rows that go wrong: the bits of ``*flags`` of each
entry point, on each of the kernels that may take the call, beside which rows
become NaN; and a session's errors."""
import numpy as np
import pytest

from detllm_b200 import synth as S

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
NONFINITE, BAD_TOKEN = 2, 64
OLD = 1 << 20  # a bit that was set before


@pytest.fixture(scope="module")
def env():
    import torch

    import detllm_b200 as D

    assert D.device_count() > 0 and torch.cuda.is_available(), "gpu tests need a CUDA device"
    torch.cuda.set_device(0)
    return D, torch, D.lib()


N, K = 6, 5


class Call:
    """One entry point on its own buffers, with a flags word."""

    def __init__(self, env, op, vocab, dtype):
        self.op, self.vocab = op, vocab
        self.lib, torch = env[2], env[1]
        self.torch = torch
        self.code = {"float32": 0, "float16": 1, "bfloat16": 2}[dtype]
        g = torch.Generator(device="cuda").manual_seed(vocab)
        self.x = torch.randn(N, vocab, generator=g, device="cuda").to(getattr(torch, dtype))
        self.tokens = torch.randint(0, vocab, (N,), generator=g, device="cuda")
        self.ids = torch.randint(0, vocab, (N, K), generator=g, device="cuda")
        self.u = torch.randn(N, K, generator=g, device="cuda")
        self.one = torch.ones(N, device="cuda")
        self.flags = torch.full((1,), OLD, dtype=torch.int32, device="cuda")

    def __call__(self):
        torch, lib, V = self.torch, self.lib, self.vocab
        head = (self.x.data_ptr(), self.code, N, V, V)
        lists = (self.ids.data_ptr(), 8, self.u.data_ptr(), 0, K, K, 1.5)
        res, ent = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda")
        stats, grad = torch.zeros(N, 4, device="cuda"), torch.zeros_like(self.x)
        top_ids = torch.zeros(N, K, dtype=torch.int32, device="cuda")
        top = torch.zeros(N, K, device="cuda")
        step = self.op in ("step", "entropy step", "list step")
        size = lib.det_step_workspace(N, V, K) if step else lib.det_scores_workspace(self.code, N, V, K)
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        tail = (self.flags.data_ptr(), work.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        tok = (self.tokens.data_ptr(), 8)
        r, e, st, gr, one = res.data_ptr(), ent.data_ptr(), stats.data_ptr(), grad.data_ptr(), self.one.data_ptr()
        if self.op == "scores":
            code = lib.det_token_scores_device(*head, *tok, 0, r, e, st, None, None, *tail)
        elif self.op == "top":
            code = lib.det_token_scores_device(*head, *tok, K, r, e, st, top_ids.data_ptr(), top.data_ptr(), *tail)
        elif self.op == "step":
            code = lib.det_token_scores_step_device(*head, *tok, one, None, r, e, st, gr, V, *tail)
        elif self.op == "entropy step":
            code = lib.det_token_scores_step_device(*head, *tok, one, one, r, e, st, gr, V, *tail)
        elif self.op == "list":
            code = lib.det_distill_loss_device(*head, *lists, r, st, *tail)
        else:
            code = lib.det_distill_step_device(*head, *lists, one, r, st, gr, V, *tail)
        assert code == 0
        bad = torch.isnan(res)
        if step:  # the gradient is NaN in the rows whose result is, and in no others
            assert torch.equal(torch.isnan(grad).all(1), bad) and torch.equal(torch.isnan(grad).any(1), bad)
        return int(self.flags[0]), bad.nonzero()[:, 0].tolist()


SCORES, LISTS = ["scores", "top", "step", "entropy step"], ["list", "list step"]
# few short rows (one kernel where there is no top list), rows of more than 16
# segments (sums and rows, or clusters), and rows of one segment among them
SHAPES = [(500, "float32"), (30000, "bfloat16"), (40000, "float32"), (131071, "float16")]


@pytest.mark.parametrize("vocab,dtype", SHAPES)
@pytest.mark.parametrize("op", SCORES + LISTS)
def test_flags_of_rows_that_are_not_numbers(env, op, vocab, dtype):
    for value, at in ((NAN, 0), (INF, vocab - 1), (NAN, vocab // 2)):
        call = Call(env, op, vocab, dtype)
        assert call() == (OLD, [])
        call.x[2] = -INF  # nothing is left: a number all the same
        assert call() == (OLD, [])
        call.x[4, at] = value
        assert call() == (OLD | NONFINITE, [4])
        call.x[4, at] = 0.0
        assert call() == (OLD | NONFINITE, [])  # never cleared


@pytest.mark.parametrize("vocab,dtype", SHAPES)
@pytest.mark.parametrize("op", SCORES)
def test_flags_of_tokens(env, op, vocab, dtype):
    for token in (vocab, 1 << 40):
        call = Call(env, op, vocab, dtype)
        call.tokens[0] = -1
        call.tokens[1] = -(1 << 40)
        assert call() == (OLD, [])
        call.tokens[3] = token
        assert call() == (OLD | BAD_TOKEN, [3])
        call.x[5, 7] = NAN
        assert call() == (OLD | BAD_TOKEN | NONFINITE, [3, 5])


@pytest.mark.parametrize("vocab,dtype", SHAPES)
@pytest.mark.parametrize("op", LISTS)
def test_flags_of_lists(env, op, vocab, dtype):
    for what in ("id", "far id", "nan", "inf"):
        call = Call(env, op, vocab, dtype)
        call.ids[0] = -1  # no entries
        call.ids[1, 2], call.u[1, 2] = -7, NAN  # not an entry: its value is not looked at
        call.u[2, 0] = -INF  # not a valid entry
        assert call() == (OLD, [])
        if what == "id":
            call.ids[3, K - 1] = vocab
        elif what == "far id":
            call.ids[3, 0] = 1 << 40
        else:
            call.u[3, 1] = NAN if what == "nan" else INF
        assert call() == (OLD | BAD_TOKEN, [3])
        call.x[5, 7] = NAN
        assert call() == (OLD | BAD_TOKEN | NONFINITE, [3, 5])


def test_a_session_s_errors_leave_it_usable(env):
    """Refused calls and a forward that met a number that is not finite: each is
    reported, the rows of the failed forward are gone, the next forward's are
    scored as before."""
    D = env[0]
    spec = S.ModelSpec(n_layer=1, d=64, d_ff=128, n_head=2, n_head_kv=2, vocab=300, ctx=16, t_embd=S.GT_F32,
                       t_attn=S.GT_F32, t_gate_up=S.GT_F32, t_down=S.GT_F32, t_out=S.GT_F32)
    g = bytearray(S.build_gguf(spec))
    toks = np.array([1, 2, 3], np.uint32)
    m = D.Model(bytes(g))
    with m.session(8, 4) as s:
        s.forward(toks, 0)
        want = s.token_scores(toks, top=4)
        for bad, rows, code in ((300, None, 35), (1, [3], 1)):
            with pytest.raises(D.DetError) as e:
                s.token_scores(np.array([bad], np.uint32), rows)
            assert e.value.code == code
        assert all(np.array_equal(a, b) for a, b in zip(want, s.token_scores(toks, top=4)))
    m.close()
    n = 300 * 64 * 4
    g[len(g) - n - 256:len(g) - n] = np.full(64, 3e38, "<f4").tobytes()  # output_norm.weight
    m = D.Model(bytes(g))
    with m.session(8, 4) as s:
        with pytest.raises(D.DetError) as e:
            s.forward(toks, 0)
        assert e.value.code == 2
        with pytest.raises(D.DetError) as e:
            s.token_scores(toks)
        assert e.value.code == 1  # no rows
    m.close()


def test_scores_of_a_model_in_parts(env):
    """Tensor parallel sessions score as sessions on one device do."""
    D = env[0]
    spec = S.ModelSpec(n_layer=2, d=512, d_ff=1024, n_head=8, n_head_kv=4, vocab=1000, ctx=64, seed=31)
    g = S.build_gguf(spec)
    toks = S.zipf_tokens(24, 1000, seed=4)
    got = []
    for m in (D.Model(g), D.Model(g, devices=[0, 0])):
        with m.session(32, 24) as s:
            s.forward(toks, 0)
            r = s.token_scores(toks, top=9)
            got.append((*r, s.distill_loss(r[2], r[3], temperature=2.0)))
        m.close()
    assert all(np.array_equal(a, b) for a, b in zip(*got))
