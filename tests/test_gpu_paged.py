"""The paged key-value cache on the GPU: append and one-token attention against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
HALF_STEP = {BF16: 2.0 ** -8, F8: 2.0 ** -4}       # torch.finfo(t).eps / 2
F8_TINY = 2.0 ** -10                               # half the spacing of e4m3's subnormals


def _K():
    from bagel_amd import _lib
    return _lib


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, gen, std=1.0, dtype=BF16):
    return (torch.randn(shape, device=DEV, generator=gen) * std).to(dtype)


def _pool(pages, page, hkv, d, dtype, order, fill):
    """A pool of ``fill`` bytes as [pages, slots, heads, d], lying as asked in memory."""
    raw = torch.uint8 if dtype == F8 else torch.int16
    full = lambda *s: torch.full(s, fill, device=DEV, dtype=raw).view(dtype)  # noqa: E731
    if order == "slots first":
        return full(pages, page, hkv, d)
    if order == "heads first":
        return full(pages, hkv, page, d).transpose(1, 2)
    assert order == "padded"                        # part of wider rows of a larger array
    return full(pages + 1, page + 1, hkv, d + 32)[1:, 1:, :, 16:16 + d]


def _values(pool):
    """A pool's stored values in 64 bits."""
    return pool.float().double()


def _scales(hkv, dtype, gen):
    if dtype != F8:
        return None, None
    return tuple((0.5 + torch.rand(hkv, device=DEV, generator=gen)) * 0.02 for _ in range(2))


NAN_BYTES = {BF16: 0x7FC1, F8: 0x7F}


# ---- append ------------------------------------------------------------------------------------------------------------

def _rope64(x, w, cos, sin, eps):
    """(values, sum of the magnitudes of the terms) of the norm and the rotation in 64 bits."""
    d = x.shape[-1]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is None:
        return x, x.abs()
    half = torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1)
    return x * cos + half * sin, (x * cos).abs() + (half * sin).abs()


def _append_case(rows, hq, hkv, d, page, dtype, order, seed, norm=True, rope=True, with_q=True, pages=None, eps=1e-6):
    K = _K()
    gen = _gen(seed)
    pages = pages or -(-rows // page) + 2
    fill = 0x3C if dtype == F8 else 0x3C01
    kp, vp = (_pool(pages, page, hkv, d, dtype, order, fill) for _ in range(2))
    ks, vs = _scales(hkv, dtype, gen)
    wide = _normal((rows, (hq + 2 * hkv) * d + 24), gen, 1.5)
    qkv = wide[:, 8:8 + (hq + 2 * hkv) * d]
    slots = torch.randperm(pages * page, device=DEV, generator=gen)[:rows].to(torch.int32)
    if rows > 2:
        slots[rows // 2] = -1
        slots[-1] = -7
    qw, kw = ((1 + _normal((d,), gen, 0.1)) if norm else None for _ in range(2))
    cos = sin = cs = None
    if rope:
        a = torch.arange(5000, device=DEV, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
        a = torch.cat((a, a), 1)
        cos, sin = a.cos().to(BF16), a.sin().to(BF16)
        cs = torch.randint(0, 5000, (rows,), device=DEV, generator=gen, dtype=torch.int32)
    Q = torch.full((rows, hq, d), 7.0, device=DEV, dtype=BF16) if with_q else None
    want = []
    live = torch.nonzero(slots >= 0)[:, 0]
    x = qkv.double().reshape(rows, hq + 2 * hkv, d)[live]
    c, s = (t[cs[live].long()].double()[:, None] if rope else None for t in (cos, sin))
    q64, q_mag = _rope64(x[:, :hq], qw, c, s, eps)
    k64, k_mag = _rope64(x[:, hq:hq + hkv], kw, c, s, eps)
    v64 = x[:, hq + hkv:]
    before = [_values(kp).clone(), _values(vp).clone()]
    K.paged_kv_append(qkv, hq, K.PagedCache(kp, vp, ks, vs), slots, Q=Q, q_norm=qw, k_norm=kw, cos_t=cos, sin_t=sin, row_cs=cs, eps=eps)
    torch.cuda.synchronize()
    at = slots[live].long()
    # 32-bit arithmetic before the one rounding: the mean square (15 roundings, halved by the root), rsqrt, division, two
    # products of the norm, two products and a sum of the rotation, a division by the scale: below 2^-19 of the terms
    slack = 2.0 ** -19
    if with_q:
        got = Q[live].double()
        assert bool(((got - q64).abs() <= HALF_STEP[BF16] * q64.abs() + slack * q_mag).all())
        dead = torch.nonzero(slots < 0)[:, 0]
        assert bool((Q[dead] == 7.0).all())
    for pool, new, mag, scale, old in ((kp, k64, k_mag, ks, before[0]), (vp, v64, v64.abs(), vs, before[1])):
        got = _values(pool)
        mine = got.reshape(-1, hkv, d)[at] if pool.is_contiguous() else got[at // page, at % page]
        if scale is not None:
            new, mag = (new / scale.double()[:, None]).clamp(-448, 448), mag / scale.double()[:, None]
            tol = torch.maximum(HALF_STEP[F8] * new.abs(), torch.tensor(F8_TINY, device=DEV)) + slack * mag
        else:
            tol = HALF_STEP[BF16] * new.abs() + slack * mag
        assert bool(((mine - new).abs() <= tol).all())
        got[at // page, at % page] = 0
        old[at // page, at % page] = 0
        assert torch.equal(got, old), "a slot that no row names changed"


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("rows,hq,hkv,d,page,order", [
    (1, 28, 4, 128, 16, "slots first"), (1, 1, 1, 64, 8, "heads first"), (2, 14, 2, 64, 64, "padded"), (3, 9, 3, 64, 8, "slots first"),
    (33, 5, 5, 128, 32, "heads first"), (257, 28, 4, 128, 16, "padded"), (1000, 24, 1, 128, 128, "heads first"), (1237, 14, 2, 64, 16, "slots first")])
def test_append_matches_definition(rows, hq, hkv, d, page, order, dtype):
    _append_case(rows, hq, hkv, d, page, dtype, order, seed=rows)


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("norm,rope,with_q", [(False, True, True), (True, False, True), (False, False, False), (True, True, False)])
def test_append_leaves_steps_out(norm, rope, with_q, dtype):
    _append_case(41, 6, 2, 128, 16, dtype, "slots first", seed=3, norm=norm, rope=rope, with_q=with_q)
    _append_case(41, 6, 2, 64, 8, dtype, "heads first", seed=4, norm=norm, rope=rope, with_q=with_q)


def test_append_without_query_heads():
    K = _K()
    gen = _gen(1)
    kv = _normal((10, 2 * 3 * 64), gen)
    kp, vp = torch.zeros((2, 8, 3, 64), device=DEV, dtype=BF16), torch.zeros((2, 8, 3, 64), device=DEV, dtype=BF16)
    slots = torch.arange(3, 13, device=DEV, dtype=torch.int32)
    K.paged_kv_append(kv, 0, K.PagedCache(kp, vp), slots)
    assert torch.equal(kp.view(16, 3, 64)[3:13], kv.view(10, 2, 3, 64)[:, 0]) and torch.equal(vp.view(16, 3, 64)[3:13], kv.view(10, 2, 3, 64)[:, 1])
    K.paged_kv_append(kv[:0], 0, K.PagedCache(kp, vp), slots[:0])       # no rows: nothing


@pytest.mark.parametrize("d,hq,hkv", [(128, 14, 2), (64, 14, 2)])
@pytest.mark.parametrize("und_rounding", [False, True])
def test_append_equals_the_workspace_scatter(und_rounding, d, hq, hkv):
    """Queries, keys and values are bit for bit those of qk_norm_rope_kv; the queries may take the place of their source."""
    K = _K()
    gen = _gen(8)
    rows, S = 70, 128
    qkv = _normal((rows, (hq + 2 * hkv) * d), gen, 1.5)
    qw, kw = 1 + _normal((d,), gen, 0.1), 1 + _normal((d,), gen, 0.1)
    cos, sin = _normal((90, d), gen).cos(), _normal((90, d), gen).sin()
    cs = torch.randint(0, 90, (rows,), device=DEV, generator=gen, dtype=torch.int32)
    slots = torch.randperm(S, device=DEV, generator=gen)[:rows].to(torch.int32)
    Q = torch.zeros((rows, hq, d), device=DEV, dtype=BF16)
    kws, vws = torch.zeros((hkv, S, d), device=DEV, dtype=BF16), torch.zeros((hkv, d, S), device=DEV, dtype=BF16)
    K.qk_norm_rope_kv(qkv, rows, hq, hkv, d, qw, qw, kw, kw, rows, cos, sin, cs, slots, Q, kws, vws, S, 1e-6, und_rounding)
    kp, vp = torch.zeros((S // 16, 16, hkv, d), device=DEV, dtype=BF16), torch.zeros((S // 16, 16, hkv, d), device=DEV, dtype=BF16)
    mine = qkv[:, :hq * d].unflatten(1, (hq, d))
    K.paged_kv_append(qkv, hq, K.PagedCache(kp, vp), slots, Q=mine, q_norm=qw, k_norm=kw, cos_t=cos, sin_t=sin, row_cs=cs, eps=1e-6,
                      und_rounding=und_rounding)
    assert torch.equal(mine, Q)
    assert torch.equal(kp.view(S, hkv, d), kws.transpose(0, 1)) and torch.equal(vp.view(S, hkv, d), vws.permute(2, 0, 1))


def test_append_special_values():
    """e4m3: values beyond the range clamp, NaN stays NaN; bf16: both stay as they are."""
    K = _K()
    x = torch.zeros((1, 2 * 64), device=DEV, dtype=BF16)
    x[0, :6] = torch.tensor([1e6, -1e6, float("inf"), float("-inf"), float("nan"), 448.0])
    x[0, 64:70] = x[0, :6]
    one = torch.ones(1, device=DEV)
    slot = torch.tensor([5], device=DEV, dtype=torch.int32)
    kp, vp = (torch.zeros((1, 8, 1, 64), device=DEV, dtype=torch.uint8).view(F8) for _ in range(2))
    K.paged_kv_append(x, 0, K.PagedCache(kp, vp, one, one), slot)
    for t in (kp, vp):
        got = t.float()[0, 5, 0, :6].tolist()
        assert got[:4] == [448.0, -448.0, 448.0, -448.0] and math.isnan(got[4]) and got[5] == 448.0
    kp, vp = (torch.zeros((1, 8, 1, 64), device=DEV, dtype=BF16) for _ in range(2))
    K.paged_kv_append(x, 0, K.PagedCache(kp, vp), slot)
    assert torch.equal(kp[0, 5, 0].view(torch.int16)[:4], x[0, :4].view(torch.int16)) and bool(torch.isnan(vp[0, 5, 0, 4]))


def test_append_rows_that_do_not_exist():
    """A slot outside the cache or a rotation row outside its table stores nothing and shows in the queries."""
    K = _K()
    gen = _gen(2)
    hq, hkv, d = 2, 1, 64
    qkv = _normal((5, (hq + 2 * hkv) * d), gen)
    kp, vp = (torch.zeros((2, 8, hkv, d), device=DEV, dtype=BF16) for _ in range(2))
    cos, sin = torch.ones((4, d), device=DEV, dtype=BF16), torch.zeros((4, d), device=DEV, dtype=BF16)
    slots = torch.tensor([0, 16, 2, 3, 2 ** 31 - 1], device=DEV, dtype=torch.int32)
    cs = torch.tensor([0, 1, 4, -1, 0], device=DEV, dtype=torch.int32)
    Q = torch.zeros((5, hq, d), device=DEV, dtype=BF16)
    K.paged_kv_append(qkv, hq, K.PagedCache(kp, vp), slots, Q=Q, cos_t=cos, sin_t=sin, row_cs=cs)
    assert torch.isnan(Q).flatten(1).all(1).tolist() == [False, True, True, True, True]
    assert torch.equal(Q[0], qkv[0, :hq * d].view(hq, d))
    assert torch.equal(kp.view(16, hkv, d)[0, 0], qkv[0, hq * d:][:d]) and not bool(kp.view(16, -1)[1:].any()) and not bool(vp.view(16, -1)[1:].any())


# ---- attention ---------------------------------------------------------------------------------------------------------

class _Case:
    def __init__(self, lens, hq, hkv, d, page, dtype, order, seed, spare=3, pages=None, q_std=2.0, first_page=0):
        gen = self.gen = _gen(seed)
        self.K = _K()
        self.lens, self.hq, self.hkv, self.d, self.page = lens, hq, hkv, d, page
        need = [-(-n // page) for n in lens]
        pages = pages or sum(need) + 2
        self.kp, self.vp = (_pool(pages, page, hkv, d, dtype, order, NAN_BYTES[dtype]) for _ in range(2))   # free slots hold NaN
        self.ks, self.vs = _scales(hkv, dtype, gen)
        ids = (first_page + torch.randperm(pages - first_page, generator=torch.Generator().manual_seed(seed))).tolist()
        width = max(need) + spare
        self.table = torch.full((len(lens), width + 2), -12345, dtype=torch.int32)   # entries behind the last page are not read
        for r, n in enumerate(lens):
            for i in range(need[r]):
                p = ids.pop()
                self.table[r, i] = p
                m = min(page, n - i * page)
                for pool, scale in ((self.kp, self.ks), (self.vp, self.vs)):
                    x = torch.randn((m, hkv, d), device=DEV, generator=gen)
                    raw = torch.uint8 if dtype == F8 else torch.int16
                    y = (x if scale is None else (x / scale[:, None]).clamp(-448, 448)).to(dtype)
                    pool.view(raw)[p, :m] = y.view(raw)
        self.table = self.table.to(DEV)[:, :width]
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        rows = len(lens)
        self.q = _normal((rows, hq * d + 16), gen, q_std)[:, 8:8 + hq * d].unflatten(1, (hq, d))
        self.o = torch.full((rows, hq * d + 8), 3.0, device=DEV, dtype=BF16)
        self.cache = self.K.PagedCache(self.kp, self.vp, self.ks, self.vs)

    def workspace(self, bound):
        return torch.zeros(self.K.paged_decode_attention_workspace_bytes(len(self.lens), self.hq, self.hkv, self.d, bound), device=DEV, dtype=torch.uint8)

    def out(self):
        return self.o[:, :self.hq * self.d].unflatten(1, (self.hq, self.d))

    def run(self, max_kv_len=None, ws=None, scale=None):
        bound = max(self.lens) if max_kv_len is None else max_kv_len
        ws = self.workspace(bound or self.table.shape[1] * self.page) if ws is None else ws
        return self.K.paged_decode_attention(self.q, self.cache, self.table, self.kv_lens, self.out(), ws, max_kv_len=bound, softmax_scale=scale)

    def want(self, scale=None):
        """(result, sum of weight x |value|) in 64 bits."""
        rep = self.hq // self.hkv
        o = torch.zeros((len(self.lens), self.hq, self.d), device=DEV, dtype=torch.float64)
        mag = o.clone()
        for r, n in enumerate(self.kv_lens.tolist()):
            if n <= 0:
                continue
            at = torch.arange(n, device=DEV)
            pages = self.table[r].long()[at // self.page]
            raw = torch.uint8 if self.kp.dtype == F8 else torch.int16
            k, v = (pool.view(raw)[pages, at % self.page].view(pool.dtype).float().double() for pool in (self.kp, self.vp))
            if self.ks is not None:
                k, v = k * self.ks.double()[:, None], v * self.vs.double()[:, None]
            for h in range(self.hkv):
                mine = slice(h * rep, (h + 1) * rep)
                p = torch.softmax(self.q[r, mine].double() @ k[:, h].t() * (scale or self.d ** -0.5), -1)
                o[r, mine], mag[r, mine] = p @ v[:, h], p @ v[:, h].abs()
        return o, mag

    def check(self, scale=None, rows=None):
        want, mag = self.want(scale)
        got = self.out().double()
        # the result's rounding to bf16 and the weights' (both half a step); scores in fp32: 128 products of size 2 x 1 and
        # their sums, times the scale, change a weight by less than 2^-12 of it
        tol = HALF_STEP[BF16] * want.abs() + (HALF_STEP[BF16] * (1 + HALF_STEP[BF16]) + 2.0 ** -12) * mag
        ok = ((got - want).abs() <= tol).flatten(1).all(1)
        rows = list(range(len(self.lens))) if rows is None else rows
        assert bool(ok[rows].all()), [(r, self.lens[r]) for r in rows if not bool(ok[r])]
        assert bool((self.o[:, self.hq * self.d:] == 3.0).all())


RAGGED = [1, 0, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 513, 1000]


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("hq,hkv,d,page,order", [
    (28, 4, 128, 16, "slots first"), (14, 2, 64, 64, "heads first"), (14, 2, 128, 8, "padded"), (9, 3, 64, 8, "slots first"),
    (16, 16, 64, 32, "heads first"), (24, 1, 128, 256, "slots first"), (40, 1, 64, 16, "padded"), (1, 1, 128, 1024, "slots first")])
def test_attention_matches_definition(hq, hkv, d, page, order, dtype):
    c = _Case(RAGGED, hq, hkv, d, page, dtype, order, seed=hq)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("n", [1, 8, 300, 1999, 4096, 70001])
@pytest.mark.parametrize("hq,hkv,d,page", [(28, 4, 128, 16), (7, 1, 64, 64)])
def test_attention_of_one_row(n, hq, hkv, d, page, dtype):
    """Alone in its launch a row is split as far as its length allows; two launches on one workspace, the tickets back at zero."""
    c = _Case([n], hq, hkv, d, page, dtype, "slots first", seed=n)
    ws = c.workspace(n)
    first = c.run(ws=ws).clone()
    c.check()
    c.o[:, :hq * d] = float("nan")
    assert torch.equal(c.run(ws=ws), first)
    assert not bool(ws[:256].any())


@pytest.mark.parametrize("bound", [0, 1, 300, 100000])
def test_attention_bound_costs_time_only(bound):
    c = _Case([5000, 3, 0, 777], 14, 2, 64, 32, BF16, "slots first", seed=5, spare=40)
    c.run(max_kv_len=bound)
    c.check()


def test_attention_scale_and_large_scores():
    c = _Case([300, 40], 8, 2, 128, 16, BF16, "slots first", seed=6)
    c.run(scale=0.31)
    # scores of 0.31 x 128 products: their fp32 error grows with the scale, 4 times that of 1 / sqrt(128)
    want, mag = c.want(0.31)
    assert bool(((c.out().double() - want).abs() <= HALF_STEP[BF16] * want.abs() + (HALF_STEP[BF16] * 1.01 + 2.0 ** -10) * mag).all())
    # one key far above the rest, in the first, a middle and the last place: the running maximum jumps
    for at in (0, 150, 299):
        c = _Case([300], 8, 2, 128, 16, BF16, "slots first", seed=7)
        page = int(c.table[0, at // 16])
        c.kp[page, at % 16] = (c.q[0, ::4] * 8).to(BF16)
        c.run()
        want, mag = c.want()
        # the scores reach 8 x 4 x 128 / sqrt(128) = 360: 128 products, each sum off by 2^-24 of it, change a weight by 2^-9
        assert bool(((c.out().double() - want).abs() <= HALF_STEP[BF16] * want.abs() + (HALF_STEP[BF16] * 1.01 + 2.0 ** -9) * mag).all())


def test_attention_shared_pages():
    """Rows that share a prefix name the same pages."""
    c = _Case([200, 200, 137], 14, 2, 64, 8, BF16, "slots first", seed=9)
    c.table[1, :20] = c.table[0, :20]
    c.table[2, :10] = c.table[0, :10]
    c.run()
    c.check()


def test_attention_pages_that_do_not_exist():
    """A page id outside the pool and a length beyond the table give NaN in their rows and leave the others alone."""
    c = _Case([100, 100, 100, 100], 14, 2, 64, 16, BF16, "slots first", seed=10)
    c.table[0, 3] = c.kp.shape[0]
    c.table[1, 6] = -1
    c.kv_lens[2] = c.table.shape[1] * 16 + 1
    c.run()
    got = torch.isnan(c.out()).flatten(1)
    assert got.all(1).tolist() == [True, True, True, False]
    assert not bool(got[3].any())
    c.lens = [0, 0, 0, 100]
    c.kv_lens[:3] = 0
    want, mag = c.want()
    assert bool(((c.out()[3].double() - want[3]).abs() <= 2.0 ** -8 * want[3].abs() + 2.0 ** -7 * mag[3]).all())


def test_attention_nan_reaches_its_heads_only():
    c = _Case([50, 50], 4, 2, 64, 16, BF16, "slots first", seed=11)
    c.kp[int(c.table[0, 1]), 3, 1, 5] = float("nan")
    c.vp[int(c.table[1, 0]), 0, 0, 7] = float("inf")
    c.run()
    out = c.out()
    assert bool(torch.isnan(out[0, 2:]).all()) and bool(torch.isfinite(out[0, :2]).all())
    assert bool(torch.isinf(out[1, :2, 7]).all()) and bool(torch.isfinite(out[1, 2:]).all()) and bool(torch.isfinite(out[1, :2, :7]).all())


@pytest.mark.parametrize("rows,n", [(1, 2500), (1, 33000), (300, 400)])
def test_attention_keys_of_infinite_scores(rows, n):
    """Scores of -inf weigh nothing, where they fill a tile, a wave's share or a chunk too; a row of nothing else is 0 / 0."""
    c = _Case([n - 17 * (i % 8) for i in range(rows)], 14, 2, 64, 16, BF16, "slots first", seed=12)
    c.q[:, :, 0] = 1.0
    at = torch.arange(n, device=DEV)
    for r, length in enumerate(c.lens[:8]):
        # from the first rows' ends backwards 1, 65, ... keys, or the first ones, or all but one in the middle
        masked = at[:length]
        masked = {0: masked[length // 2 + 1:], 1: masked[-1:], 2: masked[-65:], 3: masked[:-1], 4: masked[:300], 5: masked[masked != 130],
                  6: masked, 7: masked[128:192]}[r]
        c.kp[c.table[r].long()[masked // 16], masked % 16, :, 0] = float("-inf")
    c.run()
    if rows > 6:
        assert bool(torch.isnan(c.out()[6]).all())
    c.check(rows=[r for r in range(rows) if r != 6])


@pytest.mark.parametrize("dtype,hkv", [(BF16, 4), (F8, 8)])
def test_attention_and_append_past_32_bits(dtype, hkv):
    """A pool of more than 2^32 bytes: pages at its far end are written and read."""
    page, d = 64, 128
    pages = 2 ** 32 // (page * hkv * d * (1 if dtype == F8 else 2)) + 40
    K = _K()
    raw = torch.uint8 if dtype == F8 else torch.int16
    kp, vp = (torch.empty((pages, page, hkv, d), device=DEV, dtype=raw).view(dtype) for _ in range(2))
    gen = _gen(12)
    ks, vs = _scales(hkv, dtype, gen)
    cache = K.PagedCache(kp, vp, ks, vs)
    table = torch.tensor([[pages - 1, 0, pages - 30]], dtype=torch.int32, device=DEV)
    n = 3 * page - 5
    at = torch.arange(n, device=DEV)
    slots = (table[0, (at // page)] * page + (at % page)).to(torch.int32)
    kv = _normal((n, 2 * hkv * d), gen)
    K.paged_kv_append(kv, 0, cache, slots)
    q = _normal((1, 2 * hkv, d), gen, 2.0)
    o = torch.empty_like(q)
    ws = torch.zeros(K.paged_decode_attention_workspace_bytes(1, 2 * hkv, hkv, d, n), device=DEV, dtype=torch.uint8)
    K.paged_decode_attention(q, cache, table, torch.tensor([n], dtype=torch.int32, device=DEV), o, ws, max_kv_len=n)
    k, v = kv.double().view(n, 2, hkv, d).unbind(1)
    if dtype == F8:
        k, v = ((x / s.double()[:, None]).float().to(F8).float().double() * s.double()[:, None] for x, s in ((k, ks), (v, vs)))
    for h in range(hkv):
        p = torch.softmax(q[0, 2 * h:2 * h + 2].double() @ k[:, h].t() * d ** -0.5, -1)
        want, mag = p @ v[:, h], p @ v[:, h].abs()
        # e4m3: the quotient is rounded to 32 bits on either side, so a value on the border of two steps may be either
        # (a step is 2^-3 of it): one such value among the keys moves the result by its weight x 2^-3
        border = (p.amax(-1, keepdim=True) * v[:, h].abs().amax() * 2.0 ** -3) if dtype == F8 else 0.0
        assert bool(((o[0, 2 * h:2 * h + 2].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 * 1.01 + 2.0 ** -12) * mag + border).all())


def test_attention_captured_and_on_another_stream():
    """A captured step (append, then attention) replayed while its lengths, slots and inputs change between the replays."""
    K = _K()
    gen = _gen(13)
    hq, hkv, d, page, rows = 14, 2, 64, 16, 3
    kp, vp = (torch.zeros((64, page, hkv, d), device=DEV, dtype=BF16) for _ in range(2))
    cache = K.PagedCache(kp, vp)
    table = torch.randperm(64, device=DEV, generator=gen)[:60].view(rows, 20).to(torch.int32)
    qkv = torch.zeros((rows, (hq + 2 * hkv) * d), device=DEV, dtype=BF16)
    q, o = torch.zeros((rows, hq, d), device=DEV, dtype=BF16), torch.zeros((rows, hq, d), device=DEV, dtype=BF16)
    slots, lens = torch.full((rows,), -1, device=DEV, dtype=torch.int32), torch.zeros(rows, device=DEV, dtype=torch.int32)
    ws = torch.zeros(K.paged_decode_attention_workspace_bytes(rows, hq, hkv, d, 320), device=DEV, dtype=torch.uint8)

    def step():
        K.paged_kv_append(qkv, hq, cache, slots, Q=q)
        K.paged_decode_attention(q, cache, table, lens, o, ws, max_kv_len=320)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert not bool(o.any())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    k64, v64 = torch.zeros((rows, 320, hkv, d), device=DEV, dtype=torch.float64), torch.zeros((rows, 320, hkv, d), device=DEV, dtype=torch.float64)
    for t in range(6):
        new = [0, 299, 17][t % 3] if t < 3 else t - 2
        qkv.copy_(_normal(qkv.shape, gen))
        at = torch.tensor([new, min(new + 1, 319), 5 + t], device=DEV)
        slots.copy_(table[torch.arange(rows, device=DEV), at // page] * page + at % page)
        lens.copy_(at + 1)
        x = qkv.double().view(rows, hq + 2 * hkv, d)
        k64[torch.arange(rows), at], v64[torch.arange(rows), at] = x[:, hq:hq + hkv], x[:, hq + hkv:]
        graph.replay()
        torch.cuda.synchronize()
        for r in range(rows):
            n = int(lens[r])
            for h in range(hkv):
                mine = slice(7 * h, 7 * h + 7)
                p = torch.softmax(x[r, mine] @ k64[r, :n, h].t() * d ** -0.5, -1)
                want, mag = p @ v64[r, :n, h], p @ v64[r, :n, h].abs()
                assert bool(((o[r, mine].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 * 1.01 + 2.0 ** -12) * mag).all()), (t, r)


def test_attention_workspace_serves_smaller_calls():
    """One workspace, sized for the largest call, under batches and bounds of every size: its tickets stay where they are."""
    K = _K()
    ws = torch.zeros(K.paged_decode_attention_workspace_bytes(300, 14, 2, 64, 6000), device=DEV, dtype=torch.uint8)
    for seed, lens in enumerate(([6000], [10] * 300, [700] * 64, [5999, 1], [40] * 200 + [3000] * 20, [2500] * 7, [6000], [300] * 300)):
        c = _Case(lens, 14, 2, 64, 64, BF16, "slots first", seed=20 + seed)
        c.run(ws=ws)
        c.check()


@pytest.mark.parametrize("n,rows,hq,hkv,d,dtype", [(33000, 1, 4, 1, 128, BF16), (4500, 2, 32, 1, 64, F8), (20000, 3, 17, 1, 64, BF16)])
def test_attention_joins_in_groups(n, rows, hq, hkv, d, dtype):
    """More chunks than are joined at once, up to all that a row may have, for one and for two blocks of heads."""
    c = _Case([n - 777 * i for i in range(rows)], hq, hkv, d, 32, dtype, "slots first", seed=n)
    ws = c.workspace(n)
    first = c.run(ws=ws).clone()
    c.check()
    assert torch.equal(c.run(ws=ws), first) and not bool(ws[:16384].any())


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (6, 3, 64), (17, 1, 64)])
@pytest.mark.parametrize("lens", [[2, 0, 64, 130, 1000, 5000], [33000]])
def test_attention_keeps_the_weights_bits(lens, hq, hkv, d, dtype):
    """Values that nearly cancel show the rounding of the weights: every second key weighs a little less than the one before it
    and has its value with the other sign, so that a head's result is a small difference of two large sums."""
    c = _Case(lens, hq, hkv, d, 16, dtype, "slots first", seed=31)
    a = (1 + torch.rand((hkv, d), device=DEV, generator=c.gen) * 15).to(F8).float()         # numbers of either type
    for r, n in enumerate(lens):
        at = torch.arange(n, device=DEV)
        pages, slots = c.table[r].long()[at // 16], at % 16
        k = torch.zeros((n, hkv, d), device=DEV)
        k[::2, :, 0] = 1.0
        v = torch.where((at % 2 == 0)[:, None, None], a, -a)
        raw = torch.uint8 if dtype == F8 else torch.int16
        for pool, x in ((c.kp, k), (c.vp, v)):
            pool.view(raw)[pages, slots] = x.to(dtype).view(raw)
    step = 1.0 if c.ks is None else float(c.ks.min())
    c.q.zero_()
    c.q[:, :, 0] = ((0.01 + 0.4 * torch.rand(c.q.shape[:2], device=DEV, generator=c.gen)) * d ** 0.5 / step).to(BF16)
    c.run()
    want, mag = c.want()
    # a score is one product, below 1.3: in 32 bits with its scale off by less than 2^-21, and so is the exponential; the weights
    # as two bf16 parts are off by half a step of the second (2^-8), which is a step of the first at most (2^-7); sums and the
    # scale of the values by less than 2^-19
    tol = HALF_STEP[BF16] * want.abs() + (2.0 ** -15 + 2.0 ** -18) * mag
    got = c.out().double()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / mag.clamp(min=1e-9)).max())


def test_attention_of_infinite_values():
    """An infinite value makes its element infinite and no other, whatever its weight: a whole one, a single key's or a small one."""
    n = 96
    c = _Case([n] * n, 4, 2, 64, 16, BF16, "slots first", seed=32)
    c.table[:, :n // 16] = torch.arange(n * n // 16, device=DEV, dtype=torch.int32).view(n, -1)     # every page is some row's
    c.kp.copy_(_normal(c.kp.shape, c.gen))
    c.vp.copy_(_normal(c.vp.shape, c.gen))
    c.q.copy_(_normal(c.q.shape, c.gen, 0.5))
    c.q[::3] = 0.0                                                   # every weight 1
    want = torch.zeros((n, 4, 64), device=DEV)
    for r in range(n):
        sign = -1.0 if r % 2 else 1.0
        c.vp[int(c.table[r, r // 16]), r % 16, 1, r % 64] = sign * math.inf
        want[r, 2:, r % 64] = sign * math.inf
    c.run()
    got = c.out().float()
    assert torch.equal(torch.where(torch.isfinite(got), 0.0, got), want)


# Rows from which four heads share a thread: 1024 workgroups of 16 (head_dim 128) or 32 (64) groups of four heads, ten times as many in e4m3
@pytest.mark.parametrize("rows,hq,hkv,d,page,dtype,order,change", [
    (1900, 28, 4, 128, 16, BF16, "heads first", dict()),                               # whole groups
    (2500, 24, 1, 128, 64, BF16, "slots first", dict()),                               # keys begin and end a group, the last is of two
    (6700, 14, 2, 64, 16, BF16, "padded", dict()),                                     # queries and keys share a group, so do keys and values
    (8300, 9, 3, 64, 8, BF16, "slots first", dict()),                                  # three heads in the last group
    (8300, 9, 3, 64, 8, BF16, "slots first", dict(norm=False)), (8300, 9, 3, 64, 8, BF16, "slots first", dict(rope=False)),
    (22000, 0, 3, 64, 16, BF16, "slots first", dict(with_q=False)), (33500, 5, 2, 64, 16, BF16, "heads first", dict(with_q=False)),
    (23500, 24, 1, 128, 64, F8, "heads first", dict()), (25000, 21, 3, 128, 16, F8, "slots first", dict(norm=False)),
    (83000, 9, 3, 64, 16, F8, "padded", dict()), (66500, 14, 2, 64, 128, F8, "heads first", dict(rope=False)),
    (82500, 0, 8, 64, 128, F8, "slots first", dict(with_q=False))])
def test_append_of_many_rows(rows, hq, hkv, d, page, dtype, order, change):
    _append_case(rows, hq, hkv, d, page, dtype, order, seed=rows, **change)


@pytest.mark.parametrize("rows,d,hq,hkv", [(3400, 128, 14, 2), (8300, 64, 9, 3)])
@pytest.mark.parametrize("und_rounding", [False, True])
def test_append_of_many_rows_in_place(und_rounding, rows, d, hq, hkv):
    """Queries take the place of their source, bit for bit those of the workspace's scatter, as keys and values are."""
    K = _K()
    gen = _gen(9)
    S = -(-rows // 64) * 64
    qkv = _normal((rows, (hq + 2 * hkv) * d), gen, 1.5)
    qw, kw = 1 + _normal((d,), gen, 0.1), 1 + _normal((d,), gen, 0.1)
    cos, sin = _normal((90, d), gen).cos(), _normal((90, d), gen).sin()
    cs = torch.randint(0, 90, (rows,), device=DEV, generator=gen, dtype=torch.int32)
    slots = torch.randperm(S, device=DEV, generator=gen)[:rows].to(torch.int32)
    Q = torch.zeros((rows, hq, d), device=DEV, dtype=BF16)
    kws, vws = torch.zeros((hkv, S, d), device=DEV, dtype=BF16), torch.zeros((hkv, d, S), device=DEV, dtype=BF16)
    K.qk_norm_rope_kv(qkv, rows, hq, hkv, d, qw, qw, kw, kw, rows, cos, sin, cs, slots, Q, kws, vws, S, 1e-6, und_rounding)
    kp, vp = (torch.zeros((S // 64, 64, hkv, d), device=DEV, dtype=BF16) for _ in range(2))
    mine = qkv[:, :hq * d].unflatten(1, (hq, d))
    K.paged_kv_append(qkv, hq, K.PagedCache(kp, vp), slots, Q=mine, q_norm=qw, k_norm=kw, cos_t=cos, sin_t=sin, row_cs=cs, eps=1e-6,
                      und_rounding=und_rounding)
    assert torch.equal(mine, Q)
    assert torch.equal(kp.view(S, hkv, d), kws.transpose(0, 1)) and torch.equal(vp.view(S, hkv, d), vws.permute(2, 0, 1))


def test_append_of_many_rows_that_do_not_exist():
    K = _K()
    gen = _gen(14)
    rows, hq, hkv, d, page = 8300, 9, 3, 64, 16
    qkv = _normal((rows, (hq + 2 * hkv) * d), gen)
    pages = rows // page + 1
    kp, vp = (torch.zeros((pages, page, hkv, d), device=DEV, dtype=BF16) for _ in range(2))
    cos, sin = torch.ones((4, d), device=DEV, dtype=BF16), torch.zeros((4, d), device=DEV, dtype=BF16)
    slots, cs = torch.arange(rows, device=DEV, dtype=torch.int32), torch.arange(rows, device=DEV, dtype=torch.int32) % 4
    bad = torch.rand(rows, device=DEV, generator=gen) < 0.3
    kind = torch.arange(rows, device=DEV) % 4
    slots[bad & (kind == 0)] = pages * page
    slots[bad & (kind == 1)] = 2 ** 31 - 1
    cs[bad & (kind == 2)] = 4
    cs[bad & (kind == 3)] = -1
    Q = torch.zeros((rows, hq, d), device=DEV, dtype=BF16)
    K.paged_kv_append(qkv, hq, K.PagedCache(kp, vp), slots, Q=Q, cos_t=cos, sin_t=sin, row_cs=cs)
    x = qkv.view(rows, hq + 2 * hkv, d)
    assert torch.equal(torch.isnan(Q).flatten(1).all(1), bad) and torch.equal(Q[~bad], x[~bad, :hq])
    for pool, new in ((kp, x[:, hq:hq + hkv]), (vp, x[:, hq + hkv:])):
        assert torch.equal(pool.view(-1, hkv, d)[:rows], torch.where(bad[:, None, None], 0.0, new).to(BF16))
