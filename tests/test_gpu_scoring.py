"""Token scores and distillation on the GPU against a plain restatement in 64
bits, with the error bounds of the kernels' arithmetic.

Bounds, u = 2^-24, p the row's distribution, d_j = (x_j - m) / T, mu = sum p
|d|, k2 = sum p d^2.  An f32 power 2^y is off by 7.1 u (approximation 3.6 u, g = f + B and
its square 1.2 u, the add of D u, table 0.5 u, product 0.8 u at least); its
argument y = d log2(e) by 3 u |d| (a subtraction, the rounded log2(e) / T,
a product).  A sum adds 16 entries in a chain, 8 partial sums in a tree of
depth 3, 32 lanes in one of depth 5, and joins up to 128 segments in chains of
4 and a tree of depth 5, with a factor that is off by 7.1 u + 3 u |d| and two
roundings:

  S        relative  rs = (7.1 + 16 + 3 + 5 + 7.1 + 2 + 4 + 5) u + 6 u mu
  S1 / S   absolute  (rs + 53 u) mu + 6 u k2   (roundings of a product and of ln 2)
  log S    absolute  rs (the logarithm itself is in 64 bits)

Probabilities below 2^-123 (1e-37) of the largest count as 0: below every f32
rounding of a sum that is at least 1.
"""
import numpy as np
import pytest

from detllm_b200 import synth as S

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module")
def env():
    import torch

    import detllm_b200 as D
    from detllm_b200 import scoring

    assert D.device_count() > 0 and torch.cuda.is_available(), "gpu tests need a CUDA device"
    torch.cuda.set_device(0)
    return D, torch, scoring


# ---- the operators in 64 bits --------------------------------------------------------


def row_sums(torch, x, t=1.0):
    """Per row of x (f64): maximum, p, log p, d with 0 for masked entries, and
    the bounds' mu, k2; an empty row has p = 0."""
    m = x.max(1).values
    empty = m == -INF
    d = (x - torch.where(empty, torch.zeros_like(m), m)[:, None]) / t
    e = torch.exp(d)
    s = e.sum(1)
    d0 = torch.where(e == 0, torch.zeros_like(d), d)
    ls = torch.log(s)
    p = torch.where(empty[:, None], torch.zeros_like(e), e / s[:, None])
    logp = torch.where(empty[:, None], torch.full_like(d, -INF), d - ls[:, None])
    mu, k2 = -(p * d0).sum(1), (p * d0 * d0).sum(1)
    rs = (49.2 + 6 * mu) * U
    return dict(m=m, empty=empty, d=d0, s=s, ls=ls, p=p, logp=logp, mu=mu, k2=k2, rs=rs,
                rm=(rs + 53 * U) * mu + 6 * U * k2, s1=(e * d0).sum(1))


def scores_ref(torch, x, tokens):
    r = row_sums(torch, x)
    lp = r["logp"].gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    lp = torch.where(tokens < 0, torch.zeros_like(lp), lp)
    h = torch.where(r["empty"], torch.zeros_like(lp), r["ls"] + r["mu"])
    tol_lp = r["rs"] + U * lp.abs().nan_to_num(posinf=0) + 1e-14
    tol_h = r["rs"] + r["rm"] + U * h + 1e-14
    return r, lp, h, tol_lp, tol_h


def scores_grad_ref(torch, x, tokens, gl, gh, dtype):
    r, lp, h, _, _ = scores_ref(torch, x, tokens)
    n, _ = x.shape
    z = torch.zeros(n, dtype=torch.float64, device=x.device)
    dead = r["empty"]
    gl = torch.where(dead | (tokens < 0), z, gl.double()) if gl is not None else z
    gh = torch.where(dead, z, gh.double()) if gh is not None else z
    p, d = r["p"], r["d"]
    grad = -gl[:, None] * p - gh[:, None] * p * (d + r["mu"][:, None])
    hit = torch.zeros_like(p).scatter_(1, tokens.clamp(min=0)[:, None], gl[:, None])
    grad = grad + hit
    # dx = exp(d) (a + b d) with a = (-gl + gh S1 / S) / S, b = -gh / S
    amp = gl.abs()[:, None] + gh.abs()[:, None] * (r["mu"][:, None] + d.abs())
    tol = p * amp * (r["rs"][:, None] + (21 + 3 * d.abs()) * U) + p * (gh.abs() * r["rm"])[:, None]
    tol = tol + U * grad.abs() + type_tol(torch, grad, dtype) + 1e-37
    return grad, tol


def type_tol(torch, v, dtype):
    """Half a step of the type at v, and of its subnormals."""
    if dtype == torch.float32:
        return v.abs() * U + 2.0 ** -149
    return v.abs() * (torch.finfo(dtype).eps / 2) * (1 + 1e-3) + {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]


def teacher_ref(torch, ids, u, t):
    valid = (ids >= 0) & (u > -INF)
    some = valid.any(1)
    w = torch.where(valid, u.double() / t, torch.full_like(u, -INF, dtype=torch.float64))
    top = torch.where(some, w.max(1).values, torch.zeros(len(w), dtype=torch.float64, device=w.device))
    du = w - top[:, None]
    s = torch.where(some, torch.exp(du).sum(1), torch.ones_like(top))
    q = torch.exp(du) / s[:, None]
    logq = du - torch.log(s)[:, None]
    # an f32 power, a tree of depth 5 and a chain of 8 in f32, one division;
    # three roundings in its argument, one of them in log q too
    rq = (7.1 + 5 + 8 + 7.1 + 2 + 4 * torch.where(q > 0, du, torch.zeros_like(du)).abs().amax(1)) * U
    return valid, some, q, logq, rq


def distill_ref(torch, x, ids, u, t):
    r = row_sums(torch, x, t)
    valid, some, q, logq, rq = teacher_ref(torch, ids, u, t)
    logp = r["logp"].gather(1, ids.clamp(min=0).long())
    on = valid & (q > 0)
    diff = torch.where(on, logq - logp, torch.zeros_like(logp))
    loss = torch.where(on, q * diff, torch.zeros_like(q)).sum(1)
    # T is an f32 number, exact in both; q is off by rq, log q by rq, log p by rs
    tol = 2 * rq * (q * diff.abs().nan_to_num(posinf=0)).sum(1) + rq + r["rs"] + U * loss.abs().nan_to_num(posinf=0) + 1e-14
    return r, some, q, rq, torch.where(some, loss, torch.zeros_like(loss)), tol


def distill_grad_ref(torch, x, ids, u, t, g, dtype):
    r, some, q, rq, _, _ = distill_ref(torch, x, ids, u, t)
    live = some & ~r["empty"]
    gt = torch.where(live, g.double() / t, torch.zeros_like(g, dtype=torch.float64))
    qs = torch.zeros_like(r["p"]).scatter_add_(1, ids.clamp(min=0).long(), torch.where(ids >= 0, q, torch.zeros_like(q)))
    grad = gt[:, None] * (r["p"] - qs)
    # listed twice: a chain of up to 128 adds in f32
    tol = gt.abs()[:, None] * (r["p"] * (r["rs"][:, None] + (21 + 3 * r["d"].abs()) * U) + qs * (rq[:, None] + 132 * U))
    return grad, tol + U * grad.abs() + type_tol(torch, grad, dtype) + 1e-37


def top_ref(torch, x, k):
    """Ids of the k largest, equal ones by index (a stable sort)."""
    return torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]


def close(torch, got, ref, tol, what=""):
    got, ref = got.double(), ref.double()
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin), what
    assert torch.equal(got[~fin], ref[~fin]), what
    over = ((got - ref).abs() - tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()))


# ---- inputs ------------------------------------------------------------------------------


def make(torch, n, vocab, dtype, seed, pad=0, shift=0, masked=False, lift=True):
    """Rows in a wider store, starting `shift` entries into it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, vocab, generator=g, device="cuda") * 2.5
    if lift:
        at = torch.randint(0, vocab, (n, 5), generator=g, device="cuda")
        x.scatter_add_(1, at, torch.rand(n, 5, generator=g, device="cuda") * 11)
    if masked:
        x.masked_fill_(torch.rand(n, vocab, generator=g, device="cuda") < 0.5, -INF)
        x[n // 2] = -INF
        x[n - 1, 1:] = -INF
        x[n - 1, 0] = -3.25
    store = torch.full((n * (vocab + pad) + shift + 32,), 7.0, dtype=dtype, device="cuda")
    view = store[shift:shift + n * (vocab + pad)].view(n, vocab + pad)[:, :vocab]
    view.copy_(x)
    tokens = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    if n > 2:
        tokens[1] = -1
    return view, tokens, g


SHAPES = [  # rows, vocabulary, padding between rows, start of the first row
    (1, 1, 0, 0), (2, 2, 1, 0), (3, 7, 0, 1), (5, 31, 2, 3), (4, 128, 0, 0), (2, 255, 0, 0), (3, 257, 1, 2),
    (7, 1000, 0, 1), (3, 2047, 0, 0), (3, 2048, 8, 0), (3, 2049, 7, 5), (150, 4100, 0, 0), (1, 32000, 0, 0),
    (9, 32000, 0, 0), (2, 32768, 0, 0), (2, 32769, 0, 0), (40, 10003, 5, 0), (300, 10003, 0, 0), (3, 65537, 0, 7),
    (2, 128256, 0, 0), (2, 131072, 0, 0), (17, 131073, 0, 0), (5, 151936, 0, 0), (1, 262144, 0, 0), (2, 262143, 1, 1),
]
DTYPES = ["float32", "float16", "bfloat16"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,pad,shift", SHAPES)
def test_scores(env, n, vocab, pad, shift, dtype):
    _, torch, sc = env
    for masked in (False, True):
        x, tokens, _ = make(torch, n, vocab, getattr(torch, dtype), n + vocab, pad, shift, masked)
        xd = x.double()
        r, lp, h, tol_lp, tol_h = scores_ref(torch, xd, tokens)
        for top in sorted({0, 1, min(vocab, 20), min(vocab, 128)}):
            got = sc.token_scores(x, tokens if top % 2 else tokens.int(), top=top)
            close(torch, got.logprob, lp, tol_lp, "logprob")
            close(torch, got.entropy, h, tol_h, "entropy")
            close(torch, got.stats[:, 0], r["m"], 0 * r["m"].nan_to_num(neginf=0), "m")
            close(torch, got.stats[:, 1], r["s"] * ~r["empty"], r["s"] * r["rs"], "S")
            close(torch, got.stats[:, 2], r["s1"], r["s"] * r["rm"] + r["s1"].abs() * r["rs"], "S1")
            close(torch, got.stats[:, 3], torch.where(r["empty"], torch.full_like(lp, -INF), r["ls"]),
                  r["rs"] + U * r["ls"].abs().nan_to_num(posinf=0), "log S")
            if not top:
                assert got.top_ids is None and got.top_logprobs is None
                continue
            ids = top_ref(torch, xd, top)
            assert torch.equal(got.top_ids.long(), ids)
            best = r["logp"].gather(1, ids)
            close(torch, got.top_logprobs, best, r["rs"][:, None] + U * best.abs().nan_to_num(posinf=0) + 1e-14, "top")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,pad,shift", SHAPES)
def test_score_gradients(env, n, vocab, pad, shift, dtype):
    _, torch, sc = env
    for masked in (False, True):
        x, tokens, g = make(torch, n, vocab, getattr(torch, dtype), 3 * n + vocab, pad, shift, masked)
        gl = torch.randn(n, generator=g, device="cuda")
        gh = torch.randn(n, generator=g, device="cuda")
        xd = x.double()
        fwd = sc.token_scores(x, tokens)
        for a, b in ((gl, None), (None, gh), (gl, gh)):
            ref, tol = scores_grad_ref(torch, xd, tokens, a, b, x.dtype)
            close(torch, sc.token_scores_grad(x, tokens, fwd.stats, a, b), ref, tol, "grad")
            step, grad = sc.token_scores_step(x, tokens.int(), a, b)
            close(torch, grad, ref, tol, "step")
            assert all(torch.equal(p, q) for p, q in zip(step[:3], fwd[:3]))


LISTS = [1, 2, 8, 33, 128]


def lists(torch, x, k, g, dtype, how):
    n, vocab = x.shape
    k = min(k, vocab)
    ids = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:k] for _ in range(n)])
    u = (torch.randn(n, k, generator=g, device="cuda") * 3 + 4).to(dtype)
    if how == "ragged" and n > 1:
        ids[torch.arange(k, device="cuda")[None, :] >= torch.arange(n, device="cuda")[:, None] % (k + 1)] = -1
        u[n - 1, 0] = -INF
    if how == "twice":
        ids[:, k // 2:] = ids[:, : k - k // 2].clone()
    return ids, u


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,pad,shift", SHAPES)
def test_distillation(env, n, vocab, pad, shift, dtype):
    _, torch, sc = env
    k = LISTS[(n + vocab) % len(LISTS)]
    for i, (how, t) in enumerate([("full", 1.0), ("ragged", 2.0), ("twice", 0.625)]):
        for masked in (False, True):
            x, _, g = make(torch, n, vocab, getattr(torch, dtype), 7 * n + vocab + i, pad, shift, masked)
            ids, u = lists(torch, x, k, g, (torch.float32, torch.bfloat16, torch.float16)[i], how)
            gr = torch.randn(n, generator=g, device="cuda")
            xd = x.double()
            r, some, _, _, loss, tol = distill_ref(torch, xd, ids, u, t)
            got = sc.distill_loss(x, ids if i else ids.int(), u, t)
            close(torch, got.loss, loss, tol, "loss")
            close(torch, got.stats[:, 1], r["s"] * ~r["empty"], r["s"] * r["rs"], "S")
            ref, tolg = distill_grad_ref(torch, xd, ids, u, t, gr, x.dtype)
            close(torch, sc.distill_grad(x, ids, u, got.stats, gr, t), ref, tolg, "grad")
            step, grad = sc.distill_step(x, ids.int(), u, gr, t)
            close(torch, grad, ref, tolg, "step")
            assert torch.equal(step.loss, got.loss) and torch.equal(step.stats, got.stats)


# ---- gradients against differences ------------------------------------------------------


def test_gradients_against_differences(env):
    """Central differences of the forward calls, rows 2 j and 2 j + 1 with
    entry j moved by +h and -h.  With |f'''| <= 4 (1 + |f|) for these rows and
    values off by at most 2e-6, the difference is off by h^2 2 + 2e-6 / h."""
    _, torch, sc = env
    vocab, h, t = 60, 2.0 ** -6, 1.5
    x, _, g = make(torch, 1, vocab, torch.float32, 5)
    token = torch.tensor([17], device="cuda")
    moved = x.repeat(2 * vocab, 1)
    j = torch.arange(vocab, device="cuda")
    moved[2 * j, j] += h
    moved[2 * j + 1, j] -= h
    step = (moved[2 * j, j] - moved[2 * j + 1, j]).double()
    one = torch.ones(1, device="cuda")
    f = sc.token_scores(moved, token.repeat(2 * vocab))
    st = sc.token_scores(x, token).stats

    def diff(v):
        v = v.double()
        return (v[0::2] - v[1::2]) / step

    tol = 10 * h * h + 4e-6 / h
    lp = sc.token_scores_grad(x, token, st, one, None)[0].double()
    assert float((diff(f.logprob) - lp).abs().max()) < tol
    en = sc.token_scores_grad(x, token, st, None, one)[0].double()
    assert float((diff(f.entropy) - en).abs().max()) < tol
    ids, u = lists(torch, x, 9, g, torch.float32, "twice")
    loss = sc.distill_loss(moved, ids.repeat(2 * vocab, 1), u.repeat(2 * vocab, 1), t).loss
    grad = sc.distill_step(x, ids, u, one, t)[1][0].double()
    assert float((diff(loss) - grad).abs().max()) < tol


# ---- rows that go wrong, and ties ---------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5, 3000, 40000])
def test_rows_that_are_not_numbers(env, vocab, dtype):
    _, torch, sc = env
    x, tokens, _ = make(torch, 9, vocab, getattr(torch, dtype), vocab)
    tokens = tokens.clamp(min=0)
    x[0, vocab // 2] = float("nan")
    x[2, vocab - 1] = INF
    x[4] = INF
    x[5] = float("nan")
    x[6, 0], x[6, 1] = INF, -INF
    x[7] = -INF
    tokens[8] = vocab
    bad, fine = [0, 2, 4, 5, 6], [1, 3]
    one = torch.ones(9, device="cuda")
    k = min(vocab, 7)
    f = sc.token_scores(x, tokens, top=k)
    for v in (f.logprob, f.entropy, f.stats, f.top_logprobs):
        assert torch.isnan(v[bad]).all()
        assert torch.isfinite(v[fine]).all()
    assert (f.top_ids[bad] == -1).all() and (f.top_ids[fine] >= 0).all()
    assert f.logprob[7] == -INF and f.entropy[7] == 0 and (f.top_logprobs[7] == -INF).all()
    assert f.top_ids[7].tolist() == list(range(k))
    assert torch.isnan(f.logprob[8]) and torch.isfinite(f.entropy[8])
    for grad in (sc.token_scores_grad(x, tokens, f.stats, one, one), sc.token_scores_step(x, tokens, one, one)[1]):
        assert torch.isnan(grad[bad + [8]]).all()
        assert torch.isfinite(grad[fine]).all() and (grad[7] == 0).all()
    ids = torch.arange(k, device="cuda").repeat(9, 1)
    u = torch.randn(9, k, device="cuda")
    ids[3, 1] = vocab
    ids[1, 0], u[1, 0] = -5, float("nan")  # not an entry: its value is not looked at
    ids[5] = -1  # no list: no loss, whatever the row
    u[8, k - 1] = INF
    loss = sc.distill_loss(x, ids, u)
    step, grad = sc.distill_step(x, ids, u, one)
    again = sc.distill_grad(x, ids, u, loss.stats, one)
    assert torch.equal(step.loss.nan_to_num(nan=77), loss.loss.nan_to_num(nan=77))
    assert torch.isnan(loss.loss[[0, 2, 4, 6, 3, 8]]).all()
    assert torch.isfinite(loss.loss[1]) and loss.loss[5] == 0 and loss.loss[7] == INF
    for g in (grad, again):
        assert torch.isnan(g[[0, 2, 4, 6, 3, 8]]).all()
        assert torch.isfinite(g[1]).all() and (g[5] == 0).all() and (g[7] == 0).all()


def test_flags(env):
    D, torch, sc = env
    x, tokens, _ = make(torch, 4, 500, torch.float32, 1)
    tokens = tokens.clamp(min=0)
    out = torch.empty(4, device="cuda")
    flags = torch.full((1,), 1 << 20, dtype=torch.int32, device="cuda")

    size = D.lib().det_scores_workspace(0, 4, 500, 0)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")

    def run():
        s = torch.cuda.current_stream().cuda_stream
        assert D.lib().det_token_scores_device(x.data_ptr(), 0, 4, 500, 500, tokens.data_ptr(), 8, 0, out.data_ptr(),
                                               None, None, None, None, flags.data_ptr(), work.data_ptr(), size, s) == 0
        return int(flags[0])

    assert run() == 1 << 20
    tokens[1] = 500
    assert run() == (1 << 20) + 64
    x[2, 3] = INF
    assert run() == (1 << 20) + 64 + 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [200, 5000, 40000, 150000])
def test_ties_and_orders(env, vocab, dtype):
    """Rows whose top lists are hard to find: all equal, few values, sorted
    either way, a high stretch, fewer finite entries than the list is long."""
    _, torch, sc = env
    g = torch.Generator(device="cuda").manual_seed(vocab)
    i = torch.arange(vocab, device="cuda").float()
    rows = [torch.zeros(vocab, device="cuda"), -0.0 * (i % 2), (i % 3) - 1, i / vocab * 20, -i / vocab * 20,
            torch.where((i > vocab * 0.4) & (i < vocab * 0.4 + 9000), i * 1e-3, -5.0),
            torch.where(i % (vocab // 5 - 1) == 3, 1.0, -INF), torch.where(i == vocab - 1, -2.0, -INF),
            torch.randint(0, 9, (vocab,), generator=g, device="cuda").float(),
            torch.where(i % 700 == 9, 5.0, torch.randn(vocab, generator=g, device="cuda")),
            torch.full((vocab,), -3e38 if dtype != "float16" else -65504.0, device="cuda"),
            torch.where(i % 2 == 0, 3e38 if dtype != "float16" else 65504.0, -3e38 if dtype != "float16" else -65504.0)]
    x = torch.stack(rows).to(getattr(torch, dtype))
    tokens = torch.full((len(rows),), vocab - 1, device="cuda")
    xd = x.double()
    r, lp, h, tol_lp, tol_h = scores_ref(torch, xd, tokens)
    for top in (1, 3, 64, 128):
        f = sc.token_scores(x, tokens, top=top)
        assert torch.equal(f.top_ids.long(), top_ref(torch, xd, top)), top
        # -6e38 (the last row) is beyond f32: to nearest it is -inf, as 6e38 >
        # (2 - 2^-24) 2^127 = 3.41e38
        beyond = lp < -(2 - 2.0 ** -24) * 2.0 ** 127
        close(torch, f.logprob, torch.where(beyond, torch.full_like(lp, -INF), lp), tol_lp, "logprob")
        close(torch, f.entropy, h, tol_h, "entropy")


# ---- the same bits, whatever is around a row ----------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1003, 32000, 50000, 128256, 200001])
def test_a_row_alone_is_a_row_in_a_batch(env, vocab, dtype):
    _, torch, sc = env
    x, tokens, g = make(torch, 333, vocab, getattr(torch, dtype), vocab)
    one = torch.randn(333, generator=g, device="cuda")
    f = sc.token_scores(x, tokens, top=50)
    step, grad = sc.token_scores_step(x, tokens, one, one)
    alone = sc.token_scores_grad(x, tokens, f.stats, one, one)
    ids, u = f.top_ids, f.top_logprobs
    dl, dg = sc.distill_step(x, ids, u, one, 2.0)
    dalone = sc.distill_grad(x, ids, u, dl.stats, one, 2.0)
    assert torch.equal(dl.loss, sc.distill_loss(x, ids, u, 2.0).loss)
    assert all(torch.equal(a, b) for a, b in zip(step[:3], f[:3]))
    again = sc.token_scores(x, tokens, top=50)
    assert all(torch.equal(a, b) for a, b in zip(f, again))
    for i, n, shift, pad in ((0, 1, 0, 0), (5, 1, 3, 0), (200, 7, 1, 2), (332, 1, 5, 11), (100, 40, 0, 8)):
        store = torch.empty(n * (vocab + pad) + shift, dtype=x.dtype, device="cuda")
        y = store[shift:].view(n, vocab + pad)[:, :vocab]
        y.copy_(x[i:i + n])
        s = slice(i, i + n)
        got = sc.token_scores(y, tokens[s], top=50)
        assert all(torch.equal(a, b[s]) for a, b in zip(got, f)), (i, n)
        a, b = sc.token_scores_step(y, tokens[s], one[s], one[s])
        assert torch.equal(a.logprob, step.logprob[s]) and torch.equal(b, grad[s])
        assert torch.equal(sc.token_scores_grad(y, tokens[s], a.stats, one[s], one[s]), alone[s])
        a, b = sc.distill_step(y, ids[s], u[s], one[s], 2.0)
        assert torch.equal(a.loss, dl.loss[s]) and torch.equal(b, dg[s])
        assert torch.equal(sc.distill_grad(y, ids[s], u[s], a.stats, one[s], 2.0), dalone[s])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 300, 2049, 9001, 16385, 32768, 32769])
def test_few_rows_and_one_more(env, vocab, dtype):
    """One kernel takes as many short rows as the device holds at once, other
    kernels one row more: the same bits."""
    _, torch, sc = env
    warps = max(4, -(-vocab // 2048))
    most = 16 // warps * torch.cuda.get_device_properties(0).multi_processor_count if warps <= 16 else 5
    x, tokens, g = make(torch, most + 1, vocab, getattr(torch, dtype), vocab, 3, 1, True)
    x[2] = float("nan")
    x[3, 0] = INF
    one = torch.randn(most + 1, generator=g, device="cuda")
    k = min(vocab, 33)
    ids, u = lists(torch, x, k, g, torch.float32, "twice")

    def calls(s):
        y = x.clone()[s]
        yield from sc.token_scores(x[s], tokens[s])[:3]
        yield from sc.distill_loss(x[s], ids[s], u[s], 0.7)
        for entropy in (None, one[s]):
            a, b = sc.token_scores_step(x[s], tokens[s], one[s], entropy)
            yield from (*a[:3], b)
        a, b = sc.distill_step(y, ids[s], u[s], one[s], 0.7, out=y)
        yield from (*a, b)

    for a, b in zip(calls(slice(0, most)), calls(slice(0, most + 1)), strict=True):
        assert torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b[:most].float(), nan=1e30))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,pad,shift", [(5, 1003, 9, 1), (3, 40001, 1, 0), (200, 32000, 8, 0), (4, 151936, 5, 3)])
def test_gradient_in_place_and_beside(env, n, vocab, pad, shift, dtype):
    """Over the logits, into rows of another stride, and side by side with
    them; what lies between and around the rows stays as it was."""
    _, torch, sc = env
    dt = getattr(torch, dtype)
    x, tokens, g = make(torch, n, vocab, dt, 11, pad, shift)
    one = torch.randn(n, generator=g, device="cuda")
    ids, u = lists(torch, x, 20, g, torch.float32, "twice")
    calls = [lambda y, o: sc.token_scores_step(y, tokens, one, one, out=o)[1],
             lambda y, o: sc.token_scores_grad(y, tokens, sc.token_scores(y, tokens).stats, one, one, out=o),
             lambda y, o: sc.distill_step(y, ids, u, one, 2.0, out=o)[1],
             lambda y, o: sc.distill_grad(y, ids, u, sc.distill_loss(y, ids, u, 2.0).stats, one, 2.0, out=o)]
    for call in calls:
        want = call(x, None)
        store = torch.full((shift + n * (vocab + pad) + 40,), 3.0, dtype=dt, device="cuda")
        y = store[shift:shift + n * (vocab + pad)].view(n, vocab + pad)[:, :vocab]
        y.copy_(x)
        assert call(y, y).data_ptr() == y.data_ptr()
        assert torch.equal(y, want)
        y.fill_(3.0)
        assert bool((store == 3.0).all())
        pair = torch.full((n, 2 * vocab + 3), 3.0, dtype=dt, device="cuda")
        pair[:, 1:vocab + 1] = x
        call(pair[:, 1:vocab + 1], pair[:, vocab + 2:2 * vocab + 2])
        assert torch.equal(pair[:, 1:vocab + 1], x) and torch.equal(pair[:, vocab + 2:2 * vocab + 2], want)
        assert bool((pair[:, [0, vocab + 1, 2 * vocab + 2]] == 3.0).all())


def test_rows_far_apart(env):
    """Offsets past 2^32 entries: three rows in a store of 4.4e9 (8.8 GB)."""
    _, torch, sc = env
    vocab, ld = 5003, 2_200_000_001
    x, tokens, g = make(torch, 3, vocab, torch.float16, 3)
    store = torch.empty(2 * ld + vocab, dtype=torch.float16, device="cuda")
    far = store.as_strided((3, vocab), (ld, 1))
    far.copy_(x)
    one = torch.randn(3, generator=g, device="cuda")
    a, ga = sc.token_scores_step(x, tokens, one, one)
    b, gb = sc.token_scores_step(far, tokens, one, one, out=far)
    assert torch.equal(a.logprob, b.logprob) and torch.equal(ga, gb)
    far.copy_(x)
    f, e = sc.token_scores(x, tokens, top=9), sc.token_scores(far, tokens, top=9)
    assert all(torch.equal(p, q) for p, q in zip(f, e))
    assert torch.equal(sc.distill_step(far, f.top_ids, f.top_logprobs, one)[1],
                       sc.distill_step(x, f.top_ids, f.top_logprobs, one)[1])


def test_more_rows_than_a_grid_dimension_holds(env):
    _, torch, sc = env
    n, vocab = 66001, 19
    x, tokens, g = make(torch, n, vocab, torch.float32, 2)
    one = torch.randn(n, generator=g, device="cuda")
    fwd = sc.token_scores(x, tokens, top=2)
    _, lp, h, tol_lp, tol_h = scores_ref(torch, x.double(), tokens)
    close(torch, fwd.logprob, lp, tol_lp)
    close(torch, fwd.entropy, h, tol_h)
    ref, tol = scores_grad_ref(torch, x.double(), tokens, one, one, x.dtype)
    close(torch, sc.token_scores_grad(x, tokens, fwd.stats, one, one), ref, tol)
    close(torch, sc.token_scores_step(x, tokens, one, one)[1], ref, tol)
    ref, tol = distill_grad_ref(torch, x.double(), fwd.top_ids.long(), fwd.top_logprobs, 1.0, one, x.dtype)
    close(torch, sc.distill_step(x, fwd.top_ids, fwd.top_logprobs, one)[1], ref, tol)


def test_one_row_many_times(env):
    """An expanded row (stride 0) is read as any other."""
    _, torch, sc = env
    x, _, g = make(torch, 1, 9001, torch.bfloat16, 3)
    tokens = torch.arange(50, device="cuda")
    f = sc.token_scores(x.expand(50, 9001), tokens, top=3)
    ref = sc.token_scores(x.repeat(50, 1), tokens, top=3)
    assert all(torch.equal(a, b) for a, b in zip(f, ref))
    one = torch.ones(50, device="cuda")
    assert torch.equal(sc.token_scores_step(x.expand(50, 9001), tokens, one)[1],
                       sc.token_scores_step(x.repeat(50, 1), tokens, one)[1])


def test_no_rows(env):
    _, torch, sc = env
    x = torch.empty(0, 77, device="cuda")
    f = sc.token_scores(x, torch.empty(0, dtype=torch.int64, device="cuda"), top=5)
    assert f.logprob.shape == (0,) and f.top_ids.shape == (0, 5)
    e = torch.empty(0, device="cuda")
    l, g = sc.distill_step(x, torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, 3, device="cuda"), e)
    assert l.loss.shape == (0,) and g.shape == (0, 77)


# ---- streams and graphs ---------------------------------------------------------------------


def test_streams_and_graphs(env):
    """Two captured graphs replayed at once on two streams, with other inputs
    than they were captured with, while eager calls run on a third."""
    _, torch, sc = env
    n, vocab = 64, 50021
    sets = [make(torch, n, vocab, torch.bfloat16, s) for s in (1, 2, 3, 4)]
    one = torch.ones(n, device="cuda")

    def everything(x, tokens):
        f = sc.token_scores(x, tokens, top=30)
        step, grad = sc.token_scores_step(x, tokens, one, one)
        dl, dg = sc.distill_step(x, f.top_ids, f.top_logprobs, one, 2.0)
        return (*f, *step[:3], grad, *dl, dg)

    want = [[t.clone() for t in everything(x, tok)] for x, tok, _ in sets]
    graphs = []
    for x, tok, _ in sets[:2]:
        buf, tbuf = x.contiguous().clone(), tok.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            everything(buf, tbuf)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            out = everything(buf, tbuf)
        graphs.append((gr, s, buf, tbuf, out))
    for (gr, s, buf, tbuf, out), (x, tok, _) in zip(graphs, sets[2:]):
        buf.copy_(x)
        tbuf.copy_(tok)
    torch.cuda.synchronize()
    eager = []
    third = torch.cuda.Stream()
    for _ in range(3):
        for gr, s, *_ in graphs:
            with torch.cuda.stream(s):
                gr.replay()
        with torch.cuda.stream(third):
            eager.append(everything(sets[0][0], sets[0][1]))
    torch.cuda.synchronize()
    for (_, _, _, _, out), w in zip(graphs, want[2:]):
        assert all(torch.equal(a, b) for a, b in zip(out, w))
    for e in eager:
        assert all(torch.equal(a, b) for a, b in zip(e, want[0]))


def test_backward_of_a_user_s_own_function(env):
    """The _grad calls in an autograd function, as the module says: a captured
    backward beside an eager graph of the same leaf that is still alive."""
    _, torch, sc = env

    class CodeLength(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, tokens):
            f = sc.token_scores(x, tokens)
            ctx.save_for_backward(x, tokens, f.stats)
            return -f.logprob

        @staticmethod
        def backward(ctx, g):
            x, tokens, stats = ctx.saved_tensors
            return sc.token_scores_grad(x, tokens, stats, -g.contiguous()), None

    x, tokens, _ = make(torch, 6, 3001, torch.float32, 8)
    tokens = tokens.clamp(min=0)
    leaf = x.contiguous().clone().requires_grad_()
    CodeLength.apply(leaf, tokens).mean().backward()
    own = leaf.grad.clone()
    leaf.grad = None
    torch.nn.functional.cross_entropy(leaf.double(), tokens).backward()
    assert float((own - leaf.grad).abs().max()) < 1e-6


def test_lists_of_wider_rows_and_of_one_row(env):
    """Lists that are columns of a wider tensor; one list for every row is
    refused (its rows do not lie apart) until it is laid out."""
    D, torch, sc = env
    x, _, g = make(torch, 6, 700, torch.bfloat16, 4)
    ids = torch.randint(0, 700, (6, 40), generator=g, device="cuda")
    u = torch.randn(6, 40, generator=g, device="cuda")
    got = sc.distill_loss(x, ids[:, 3:20], u[:, 3:20], 2.0)
    want = sc.distill_loss(x, ids[:, 3:20].contiguous(), u[:, 3:20].contiguous(), 2.0)
    assert torch.equal(got.loss, want.loss)
    with pytest.raises(D.DetError):
        sc.distill_loss(x, ids[:1].expand(6, 40), u[:1].expand(6, 40))
    with pytest.raises(ValueError):
        sc.distill_loss(x, ids[:, 3:20], u[:, 3:20].contiguous())
    with pytest.raises(ValueError):
        sc.distill_loss(x.t(), ids, u)
    for top in (129, -1):
        with pytest.raises(ValueError):
            sc.token_scores(x, torch.zeros(6, dtype=torch.int64, device="cuda"), top=top)
    with pytest.raises(D.DetError):  # a gradient of nothing
        sc.token_scores_step(x, torch.zeros(6, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("t", [1e-6, 1e-3, 1e3, 1e6])
def test_extreme_temperatures(env, t):
    _, torch, sc = env
    x, _, g = make(torch, 5, 5000, torch.float32, 9)
    ids, u = lists(torch, x, 33, g, torch.float32, "full")
    gr = torch.randn(5, generator=g, device="cuda")
    t32 = float(np.float32(t))  # the library takes an f32
    _, _, _, _, loss, tol = distill_ref(torch, x.double(), ids, u, t32)
    step, grad = sc.distill_step(x, ids, u, gr, t)
    close(torch, step.loss, loss, tol, "loss")
    ref, tolg = distill_grad_ref(torch, x.double(), ids, u, t32, gr, x.dtype)
    close(torch, grad, ref, tolg, "step")
    close(torch, sc.distill_grad(x, ids, u, step.stats, gr, t), ref, tolg, "grad")


def test_one_token_in_every_entry_of_a_list(env):
    _, torch, sc = env
    x, _, g = make(torch, 3, 40000, torch.float16, 10)
    ids = torch.full((3, 128), 39999, device="cuda")
    u = torch.randn(3, 128, generator=g, device="cuda")
    gr = torch.ones(3, device="cuda")
    step, grad = sc.distill_step(x, ids, u, gr)
    _, _, _, _, loss, tol = distill_ref(torch, x.double(), ids, u, 1.0)
    close(torch, step.loss, loss, tol, "loss")
    ref, tolg = distill_grad_ref(torch, x.double(), ids, u, 1.0, gr, x.dtype)
    close(torch, grad, ref, tolg, "grad")


FIRST = """
import torch
from detllm_b200 import scoring as sc
x = torch.randn(9, 40001, device="cuda"); t = torch.randint(0, 40001, (9,), device="cuda")
g = torch.ones(9, device="cuda"); graph = torch.cuda.CUDAGraph(); torch.cuda.synchronize()
with torch.cuda.graph(graph):
    f = sc.token_scores(x, t, top=20)
    s, d = sc.token_scores_step(x, t, g)
    l, e = sc.distill_step(x, f.top_ids, f.top_logprobs, g, 2.0)
    h = sc.token_scores_grad(x, t, f.stats, g, g)
graph.replay(); torch.cuda.synchronize()
f2 = sc.token_scores(x, t, top=20)
assert all(torch.equal(a, b) for a, b in zip(f, f2))
assert torch.equal(d, sc.token_scores_step(x, t, g)[1])
assert torch.equal(e, sc.distill_step(x, f2.top_ids, f2.top_logprobs, g, 2.0)[1])
assert torch.equal(h, sc.token_scores_grad(x, t, f2.stats, g, g))
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture(env):
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_host_threads_at_once(env):
    """Calls from several host threads, each on its own stream."""
    import threading

    _, torch, sc = env
    sets = [make(torch, 40, 30011, torch.bfloat16, 20 + i) for i in range(4)]
    one = torch.ones(40, device="cuda")
    want = [(sc.token_scores(x, t, top=9), sc.token_scores_step(x, t, one, one)[1]) for x, t, _ in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        x, t, _ = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                f, d = sc.token_scores(x, t, top=9), sc.token_scores_step(x, t, one, one)[1]
            torch.cuda.current_stream().synchronize()
        if not (all(torch.equal(a, b) for a, b in zip(f, want[i][0])) and torch.equal(d, want[i][1])):
            bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


# ---- sessions, and a run of all of them together ---------------------------------------------


@pytest.fixture(scope="module")
def models(env):
    D = env[0]
    spec = dict(n_layer=2, d=256, d_ff=512, n_head=4, n_head_kv=2, vocab=1024, ctx=64)
    teacher = D.Model(S.build_gguf(S.ModelSpec(**spec, seed=11)))
    student = D.Model(S.build_gguf(S.ModelSpec(**spec, seed=12, t_attn=S.GT_Q4_0)))
    yield teacher, student
    teacher.close()
    student.close()


def test_session_scores(env, models):
    D, torch, sc = env
    m = models[0]
    toks = S.zipf_tokens(24, 1024, seed=4)
    with m.session(n_ctx=32, max_chunk=24) as s:
        logits = s.forward(toks, 0, want_logits=True)
        x = torch.from_numpy(logits).cuda()
        rows = np.array([3, 3, 0, 23, 7], np.uint32)
        want = np.array([5, 1023, 0, 77, 0xFFFFFFFF], np.uint32)
        lp, en, ids, lps = s.token_scores(want, rows, top=12)
        t = torch.from_numpy(want.astype(np.int64)).cuda()
        t[4] = -1
        f = sc.token_scores(x[torch.from_numpy(rows.astype(np.int64)).cuda()], t, top=12)
        for a, b in ((lp, f.logprob), (en, f.entropy), (ids.astype(np.int32), f.top_ids), (lps, f.top_logprobs)):
            assert np.array_equal(a, b.cpu().numpy())
        lp2, *_ = s.token_scores(toks)
        assert np.array_equal(lp2, sc.token_scores(x, torch.from_numpy(toks.astype(np.int64)).cuda()).logprob.cpu().numpy())
        # what the coder pays: freq / total, each count at least 1
        r = s.symbol_ranges(toks, byte_escapes=False).astype(np.float64)
        bits = -np.log2(r[:, 1] / r[:, 2])
        # freq = floor(p 2^24) + 1 and total = 2^24 + vocab at most: 2^-24 / p
        # + 1024 2^-24, and the f32 of both sides
        p = np.exp(lp2.astype(np.float64))
        assert np.all(np.abs(bits + lp2 / np.log(2)) < (2.0 ** -24 / p + 1024 * 2.0 ** -24 + 1e-5) / np.log(2))
        for bad, code in (((np.array([1024]), None, 0), 35), ((np.array([1]), np.array([24]), 0), 1),
                          ((np.array([1]), None, 129), 63)):
            with pytest.raises(D.DetError) as e:
                s.token_scores(bad[0], bad[1], top=bad[2])
            assert e.value.code == code
        assert s.token_scores(np.zeros(0, np.uint32))[0].size == 0
        # the ranges are as they were
        assert np.array_equal(s.symbol_ranges(toks, byte_escapes=False), r.astype(np.uint64))


def test_session_distillation(env, models):
    D, torch, sc = env
    teacher, student = models
    toks = S.zipf_tokens(24, 1024, seed=5)
    with teacher.session(32, 24) as a, student.session(32, 24) as b:
        a.forward(toks, 0)
        x = torch.from_numpy(b.forward(toks, 0, want_logits=True)).cuda()
        _, _, ids, lps = a.token_scores(toks, top=20)
        ids[4, 3:] = 0xFFFFFFFF
        loss = b.distill_loss(ids, lps, temperature=2.0)
        di, du = torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(lps).cuda()
        ref = sc.distill_loss(x, di, du, 2.0).loss
        assert np.array_equal(loss, ref.cpu().numpy()) and (loss > 0).all()
        # of the teacher's own rows: only what its list leaves out
        own = a.distill_loss(ids, lps)
        mass = np.where(ids == 0xFFFFFFFF, 0.0, np.exp(lps.astype(np.float64))).sum(1)
        assert np.allclose(own, -np.log(mass), atol=1e-5)
        for bad, code in ((1024, 35), (np.nan, 34), ("rows", 1)):
            i2, l2 = ids.copy(), lps.copy()
            if bad == 1024:
                i2[2, 2] = bad
            elif bad != "rows":
                l2[3, 1] = bad
            with pytest.raises(D.DetError) as e:
                b.distill_loss(i2, l2, np.arange(1, 25) if bad == "rows" else None)
            assert e.value.code == code


def test_score_is_what_compress_pays(env, models):
    """Model.score under the codec's windows against the payload: the codec's
    counts cost at most (2^-24 / p + vocab 2^-24) / ln 2 bits more per token,
    and its byte-wise carry and tail less than 10 bytes."""
    D = env[0]
    m = models[0]
    toks = S.zipf_tokens(400, 1024, seed=9)
    for n_ctx in (64, 40, 7):
        lp, en, ids, lps = m.score(toks, n_ctx, top=5)
        payload = m.encode_symbols(toks, n_ctx, n_ctx // 4, byte_escapes=False)
        bits = float(-lp.astype(np.float64).sum() / np.log(2))
        slack = float(((2.0 ** -24 / np.exp(lp.astype(np.float64)) + 1024 * 2.0 ** -24 + 1e-5) / np.log(2)).sum())
        assert abs(8 * len(payload) - bits) < slack + 80
        assert (ids[1:, 0] < 1024).all() and (lps[:, 0] >= lps[:, 4]).all()
    with pytest.raises(ValueError):
        m.score(toks, 65)
    with pytest.raises(ValueError):
        m.score(np.array([1, 1024]), 64)
    assert m.score(np.zeros(0, np.uint32))[0].size == 0


def test_distilling_runs_end_to_end(env, models):
    """The operators as they are used together: a teacher scores a text and
    gives its alternatives; a student's logits take steps down the distillation
    gradient, each checked against the 64-bit gradient at the same point."""
    _, torch, sc = env
    teacher, student = models
    toks = S.zipf_tokens(64, 1024, seed=6)
    x = torch.from_numpy(teacher.logits_for_tokens(toks)).cuda()
    z = torch.from_numpy(student.logits_for_tokens(toks)).cuda()
    nxt = torch.from_numpy(np.roll(toks, -1).astype(np.int64)).cuda()
    nxt[-1] = -1
    f = sc.token_scores(x, nxt, top=32)
    g = torch.full((64,), 1 / 64, device="cuda")
    for _ in range(3):
        loss, grad = sc.distill_step(z, f.top_ids, f.top_logprobs, g, 2.0)
        ref, tol = distill_grad_ref(torch, z.double(), f.top_ids.long(), f.top_logprobs, 2.0, g, z.dtype)
        close(torch, grad, ref, tol, "distill")
        code, hard = sc.token_scores_step(z, nxt, -g)
        ref, tol = scores_grad_ref(torch, z.double(), nxt, -g, None, z.dtype)
        close(torch, hard, ref, tol, "code length")
        z -= 20.0 * (grad + hard)
