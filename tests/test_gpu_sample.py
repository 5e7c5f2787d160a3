"""Sampling on the GPU against its definition: a stable sort and sums in 64 bits.  Tokens have to be equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = torch.bfloat16
INF = float("inf")


def _K():
    from bagel_amd import _lib
    return _lib


def _want(logits, u, t, k, p, m):
    """(token, logprob) of every row."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -INF, x)
    n = x.shape[1]
    x, index = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(n, device=DEV)
    u, t, k, p, m = (v.double()[:, None] for v in (u, t, k, p, m))
    greedy = ~(t > 0)
    z = torch.where(x == x[:, :1], 0.0, (x - x[:, :1]) / torch.where(greedy, 1.0, t))
    z = torch.where((x[:, :1] == INF) & (x < INF), -INF, z)       # -inf / inf is no number, but infinitely less is no weight
    w = torch.where(x == -INF, 0.0, torch.exp(z))
    w = torch.where(rank < torch.where(greedy, 1, torch.where(k <= 0, n, k)), w, 0.0)
    sums = torch.cumsum(w, -1)
    w = torch.where(~(p < 1) | (sums - w < p * sums[:, -1:]) | (rank == 0), w, 0.0)
    w = torch.where(~(m > 0) | (w >= m) | (rank == 0), w, 0.0)
    sums = torch.cumsum(w, -1)
    total = sums[:, -1:]
    last = (w > 0).double().mul(rank + 1).amax(-1, keepdim=True).long() - 1
    at = torch.minimum((sums <= u * total).sum(-1, keepdim=True), last.clamp(min=0))
    token, logprob = index.gather(1, at)[:, 0], (z.gather(1, at) - torch.log(total))[:, 0]
    none = x[:, 0] == -INF
    return torch.where(none, 0, token), torch.where(none, -INF, logprob)


def _settings(rows, gen, t=None, k=None, p=None, m=None, n=1000):
    r = lambda: torch.rand(rows, device=DEV, generator=gen)  # noqa: E731
    const = lambda v, other: other if v is None else torch.full((rows,), float(v), device=DEV)  # noqa: E731
    return dict(u=r(), t=const(t, 0.2 + 1.5 * r()), k=const(k, (r() * 1.3 * n * r() ** 4).floor()).to(torch.int32), p=const(p, (r() * 1.1).clamp(max=1.0)),
                m=const(m, r() ** 3 * 0.3))


def _check(logits, u, t, k, p, m, what=""):
    K = _K()
    rows, n = logits.shape
    ws = torch.full((K.sample_rows_workspace_bytes(rows, n),), 0xA5, device=DEV, dtype=torch.uint8)       # any content will do
    tokens = torch.full((rows,), -9, device=DEV, dtype=torch.int32)
    logprobs = torch.full((rows,), 9.0, device=DEV)
    K.sample_rows(logits, u, tokens, ws, temperature=t, top_k=k, top_p=p, min_p=m, logprobs=logprobs)
    token, logprob = _want(logits, u, t, k, p, m)
    off = torch.nonzero(tokens.long() != token)[:, 0].tolist()
    assert not off, (what, [(r, int(tokens[r]), int(token[r]), float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(m[r])) for r in off[:4]])
    # one rounding to 32 bits of a 64-bit value; weights good to 2^-32 of themselves move the logarithm of their sum below 2^-31
    fine = torch.isfinite(logprob)
    assert torch.equal(fine, torch.isfinite(logprobs)), what
    assert bool(((logprobs.double() - logprob).abs()[fine] <= 2.0 ** -24 * logprob.abs()[fine] + 2.0 ** -24).all()), what
    return tokens


def _logits(rows, n, gen, dtype, std=2.5):
    x = torch.randn((rows, n), device=DEV, generator=gen) * std
    at = torch.randint(0, n, (rows, min(n, 20)), device=DEV, generator=gen)
    x.scatter_reduce_(1, at, torch.rand(at.shape, device=DEV, generator=gen) * 16 - 2, "amax")
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (5, 7), (4, 8), (9, 9), (64, 100), (33, 1000), (20, 4095), (7, 4097), (50, 8200), (3, 40001),
                                    (40, 65536), (70, 152064), (300, 20000)])
def test_sampling_matches_definition(rows, n, dtype):
    gen = torch.Generator(device=DEV).manual_seed(rows * 7 + n)
    logits = _logits(rows, n, gen, dtype)
    for i, change in enumerate((dict(), dict(k=0, p=1.0, m=0.0), dict(k=0, m=0.0), dict(k=20, p=0.8, m=0.0, t=0.7), dict(p=1.0, m=0.0), dict(k=0, p=1.0))):
        _check(logits, **_settings(rows, gen, n=n, **change), what=f"settings {i}")


def test_sampling_without_settings_and_with_a_few():
    K = _K()
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, u = _logits(6, 5000, gen, BF16), torch.rand(6, device=DEV, generator=gen)
    ones, zeros = torch.ones(6, device=DEV), torch.zeros(6, device=DEV)
    ws = torch.empty(K.sample_rows_workspace_bytes(6, 5000), device=DEV, dtype=torch.uint8)
    tokens = torch.empty(6, device=DEV, dtype=torch.int32)
    K.sample_rows(x, u, tokens, ws)
    assert torch.equal(tokens.long(), _want(x, u, ones, zeros, ones, zeros)[0])
    K.sample_rows(x, u, tokens, ws, top_p=ones * 0.5)
    assert torch.equal(tokens.long(), _want(x, u, ones, zeros, ones * 0.5, zeros)[0])
    K.sample_rows(x[:0], u[:0], tokens[:0], ws)          # no rows: nothing


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("kind", ["equal", "few values", "two levels", "flat", "steep", "lowest", "minus infinity", "one live", "plus infinity", "nan"])
def test_sampling_of_unusual_rows(kind, dtype):
    """Ties by the thousand (the index decides), masks, infinities: each with small and large temperatures and every filter."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    rows, n = 24, 30000
    x = torch.randn((rows, n), device=DEV, generator=gen)
    if kind == "equal":
        x = torch.full_like(x, -3.0)
    elif kind == "few values":
        x = x.round()
        x[:, ::3] = -0.0
    elif kind == "two levels":
        x = torch.where(x > 1, 4.0, 1.0)
    elif kind == "flat":
        x = x * 1e-3
    elif kind == "steep":
        x = x * 1000
    else:
        low = {"lowest": torch.finfo(dtype).min, "nan": float("nan")}.get(kind, -INF)
        if kind == "one live":
            keep = torch.zeros_like(x, dtype=torch.bool)
            keep[torch.arange(rows), torch.randint(0, n, (rows,), device=DEV, generator=gen)] = True
        else:
            keep = torch.rand(x.shape, device=DEV, generator=gen) < 0.3
            keep[3] = False
        x = torch.where(keep, x, low)
        if kind == "plus infinity":
            x[:, 100:20000:77] = INF
            x[5, 17] = float("nan")
    x = x.to(dtype)
    for t in (0.01, 1.0, 30.0, 1e9, INF):
        for change in (dict(k=0, p=1.0, m=0.0), dict(k=0, m=0.0), dict(p=1.0, m=0.0), dict(k=0, p=1.0), dict()):
            _check(x, **_settings(rows, gen, t=t, n=n, **change), what=(kind, t, change))


def test_sampling_settings_at_their_ends():
    gen = torch.Generator(device=DEV).manual_seed(6)
    x = _logits(8, 9000, gen, BF16)
    base = _settings(8, gen, t=0.9, k=40, p=0.9, m=0.01)
    f = lambda *v: torch.tensor(v, device=DEV)  # noqa: E731
    first = x.float().argmax(1)
    for name, v in (("t", f(0.0, -1.0, float("nan"), 0.9, 1e-30, 1e-38, 1e30, INF)), ("k", f(0, -5, 1, 2, 8999, 9000, 9001, 2 ** 31 - 1).to(torch.int32)),
                    ("p", f(0.0, -1.0, float("nan"), 1.0, 2.0, 1e-9, 0.99999994, 0.5)), ("m", f(0.0, -1.0, float("nan"), 1.0, 1.5, INF, 1e-20, 0.5)),
                    ("u", f(0.0, 1e-30, 0.99999994, 1.0, 1.5, -1.0, INF, 0.5))):
        s = dict(base, **{name: v})
        want = dict(s)
        if name == "u":
            want["u"] = v.clamp(0, 1)
        if name == "p":
            want["p"] = torch.where(torch.isnan(v), 1.0, v)
        K = _K()
        ws = torch.zeros(K.sample_rows_workspace_bytes(8, 9000), device=DEV, dtype=torch.uint8)
        tokens = torch.empty(8, device=DEV, dtype=torch.int32)
        K.sample_rows(x, s["u"], tokens, ws, temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
        assert torch.equal(tokens.long(), _want(x, **want)[0]), name
        if name == "t":
            assert torch.equal(tokens.long()[:3], first[:3])
    nan_u = torch.full((8,), float("nan"), device=DEV)
    K.sample_rows(x, nan_u, tokens, ws, temperature=base["t"])
    assert torch.equal(tokens.long(), first)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_sampling_strides(dtype):
    """Rows of a wider array, at odd addresses, and one row of logits for many draws."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    wide = _logits(10, 20011, gen, dtype)
    _check(wide[:, 1:20002], **_settings(10, gen))
    _check(wide[::2, 8:20000], **_settings(5, gen))
    _check(wide[3:4].expand(50, -1), **_settings(50, gen))
    _check(wide[4:5, 3:77].expand(50, -1), **_settings(50, gen, n=74))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_sampling_of_rows_at_every_address(dtype):
    """A vocabulary of odd size puts its rows on every boundary; so do views that begin inside a row."""
    gen = torch.Generator(device=DEV).manual_seed(17)
    for n in (1, 3, 9, 8191, 8193, 16385, 33333):
        _check(_logits(9, n, gen, dtype), **_settings(9, gen, n=n), what=n)
        _check(_logits(9, n, gen, dtype), **_settings(9, gen, n=n, k=0, p=1.0, m=0.0), what=n)
    flat = _logits(1, 40000, gen, dtype)[0]
    for first in range(1, 9):
        for n in (5, 8192 - first, 8192, 20000):
            x = flat[first:first + n][None]
            x[0, -1] = 30.0                                  # the last one of the row, and what lies beyond it, count or not
            _check(x, **_settings(1, gen, n=n), what=(first, n))
    x = torch.full((6, 70001), -INF, device=DEV).to(dtype)
    _check(x, **_settings(6, gen, t=0.0), what="nothing")
    _check(x, **_settings(6, gen), what="nothing")


def test_sampling_of_the_largest_row():
    gen = torch.Generator(device=DEV).manual_seed(18)
    n = 1 << 20
    wide = _logits(2, n + 3, gen, BF16)
    _check(wide[:, 1:n + 1], **_settings(2, gen, n=n))
    _check(wide[:, :n], **_settings(2, gen, n=n, k=0, p=0.9))


def test_sampling_workspace_serves_fewer_rows():
    K = _K()
    gen = torch.Generator(device=DEV).manual_seed(19)
    n = 50001
    ws = torch.full((K.sample_rows_workspace_bytes(70, n),), 0x77, device=DEV, dtype=torch.uint8)
    for rows in (70, 1, 13, 64, 33):
        x, s = _logits(rows, n, gen, BF16), _settings(rows, gen, n=n)
        tokens = torch.empty(rows, device=DEV, dtype=torch.int32)
        K.sample_rows(x, s["u"], tokens, ws, temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
        assert torch.equal(tokens.long(), _want(x, **s)[0])


def test_sampling_does_not_depend_on_the_batch():
    gen = torch.Generator(device=DEV).manual_seed(8)
    x = _logits(64, 152064, gen, BF16)
    s = _settings(64, gen, n=152064)
    every = _check(x, **s)
    for r in (0, 31, 63):
        one = _check(x[r:r + 1], **{name: v[r:r + 1] for name, v in s.items()})
        assert int(one[0]) == int(every[r])


def test_sampling_follows_the_distribution():
    """20000 evenly spread numbers draw every kept token in proportion to its weight, to within one draw either side of the
    quotient's whole part; the others never."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = _logits(1, 300, gen, torch.float32)
    rows = 20000
    u = (torch.arange(rows, device=DEV) + 0.5) / rows
    s = dict(t=torch.full((rows,), 0.8, device=DEV), k=torch.full((rows,), 50, device=DEV, dtype=torch.int32), p=torch.full((rows,), 0.95, device=DEV),
             m=torch.zeros(rows, device=DEV))
    tokens = _check(x.expand(rows, -1), u, **s)
    seen = torch.bincount(tokens.long(), minlength=300).double()
    w = torch.softmax(x[0].double() / 0.8, 0)
    order = torch.sort(w, descending=True).indices[:50]
    w = w[order] / w[order].sum()
    kept = int((torch.cumsum(w, 0) < 0.95).sum()) + 1
    want = torch.zeros(300, device=DEV, dtype=torch.float64)
    want[order[:kept]] = w[:kept] / w[:kept].sum() * rows
    assert bool(((seen - want).abs() <= 1.0 + 1e-6 * rows).all())


def test_sampling_captured():
    K = _K()
    gen = torch.Generator(device=DEV).manual_seed(10)
    rows, n = 5, 50000
    x = _logits(rows, n, gen, BF16)
    s = _settings(rows, gen, n=n)
    ws = torch.zeros(K.sample_rows_workspace_bytes(rows, n), device=DEV, dtype=torch.uint8)
    tokens = torch.zeros(rows, device=DEV, dtype=torch.int32)
    logprobs = torch.zeros(rows, device=DEV)

    def step():
        K.sample_rows(x, s["u"], tokens, ws, temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"], logprobs=logprobs)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(6):
        x.copy_(_logits(rows, n, gen, BF16))
        for name, v in _settings(rows, gen, n=n).items():
            s[name].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        token, logprob = _want(x, **s)
        assert torch.equal(tokens.long(), token)
        assert math.isfinite(float(logprobs.sum())) and bool(((logprobs.double() - logprob).abs() <= 2.0 ** -24 * logprob.abs() + 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("change", [dict(k=0, p=1.0), dict(k=0, p=0.999), dict(k=9000, p=1.0), dict(k=9000, p=0.999)])
@pytest.mark.parametrize("n", [20000, 152064])
def test_sampling_of_the_last_token_above_min_p(n, change, dtype):
    """A uniform at or beyond 1 draws the last token that the filters keep, and none that min-p leaves out, also where min-p's
    border lies among thousands of tokens of nearly its weight."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    rows = 48
    x = torch.randn((rows, n), device=DEV, generator=gen).to(dtype)
    s = _settings(rows, gen, t=1.0, **change)
    s["m"] = 10.0 ** (-1 - 3 * torch.rand(rows, device=DEV, generator=gen))
    for u in (1.0, 3.0, INF):
        want = _want(x, torch.ones(rows, device=DEV), s["t"], s["k"], s["p"], s["m"])[0]
        K = _K()
        ws = torch.zeros(K.sample_rows_workspace_bytes(rows, n), device=DEV, dtype=torch.uint8)
        tokens = torch.empty(rows, device=DEV, dtype=torch.int32)
        K.sample_rows(x, torch.full((rows,), u, device=DEV), tokens, ws, temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
        off = torch.nonzero(tokens.long() != want)[:, 0].tolist()
        assert not off, (u, len(off), [(r, int(tokens[r]), int(want[r])) for r in off[:4]])


def _chunks(rows, n, dtype):
    """Chunks of 8192 logits per slice that a call on these sizes is cut into, from the workspace that its refusal asks for."""
    import ctypes
    import re
    K = _K()
    a = ctypes.c_void_p(1 << 20)                              # refused before it is followed
    assert K.lib().bagel_sample_rows(a, K.L(n), K.I(rows), K.I(n), K.I(int(dtype == torch.float32)), a, None, None, None, None, a, None, a, K.L(0), None)
    need = int(re.search(r"(\d+) needed", K.lib().bagel_last_error().decode()).group(1))
    slices = need // rows // (16 + 512 * 8 + 1408 * 8)        # a slice's summary, list and bins
    return [c for c in (1, 2, 3, 4) if -(-(n + 7) // (8192 * c)) == slices]


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("chunks,rows,n", [(1, 9, 60001), (2, 6, 152064), (2, 40, 65537), (3, 64, 65537), (3, 60, 152064), (4, 100, 151936), (2, 260, 32003), (4, 250, 32003),
                                           (4, 2, 1 << 20)])
def test_sampling_in_slices_of_every_size(chunks, rows, n, dtype):
    """One to four chunks per slice, rows of more than ten slices, rows off 16-byte boundaries."""
    assert chunks in _chunks(rows, n, dtype)
    gen = torch.Generator(device=DEV).manual_seed(23)
    x = _logits(rows, n + 3, gen, dtype)[:, 1:n + 1]
    for change in (dict(k=0, p=0.95, m=0.0), dict(k=20, p=0.8, m=0.0), dict(k=0, p=1.0, m=0.0), dict(t=0.0), dict()):
        _check(x, **_settings(rows, gen, n=n, **change), what=(chunks, change))
