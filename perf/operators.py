"""The operators of a paged decoding step as measured cases: the append of keys and values to a paged cache (with the
q/k norm and the rotation on the way), one new token's attention over such a cache, and the sampling of its logits.

``own = False`` computes them in their plain form, elementary torch operations in 32 bits (64 where sums meet a border);
``own = True`` makes the calls that a serving loop makes of bagel_amd's kernels.  Head layouts are those of
bagel_amd.config: 28 / 4 heads of 128 and 14 / 2 heads of 64, besides one kv head per query head and one for all.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
THETA = 1000000.0
EPS = 1e-6
F8 = torch.float8_e4m3fn
F8_MAX = 448.0


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a single conversation's step: one row's q/k norm, rotation and append, where the launch is all there is
        dict(name="append 1 row", op="append", rows=1, seqs=1, hq=28, hkv=4, d=128, page=16, f8=False, heads_first=False),
        # a step of 64 conversations into an 8-bit cache, some rows of the batch being padding
        dict(name="append 64 rows f8", op="append", rows=64, seqs=64, hq=28, hkv=4, d=128, page=64, f8=True, heads_first=False),
        # three ragged prompts prefilled together
        dict(name="append 2347 rows", op="append", rows=2347, seqs=3, hq=14, hkv=2, d=64, page=16, f8=False, heads_first=True),
        # the largest: a batch of long prompts
        dict(name="append 32768 rows", op="append", rows=32768, seqs=9, hq=28, hkv=4, d=128, page=64, f8=False, heads_first=False),
        # one conversation at an ordinary length: latency
        dict(name="attend 1 x 700", op="attend", rows=1, longest=700, hq=28, hkv=4, d=128, page=16, f8=False, heads_first=False),
        # one long document: the split over the length and its join
        dict(name="attend 1 x 131072", op="attend", rows=1, longest=131072, hq=28, hkv=4, d=128, page=64, f8=False, heads_first=False),
        # a serving batch of ragged conversations, one slot of it free (length 0)
        dict(name="attend 64 x 8192", op="attend", rows=64, longest=8192, hq=28, hkv=4, d=128, page=64, f8=False, heads_first=True),
        # the small model over an 8-bit cache
        dict(name="attend 48 x 5000 f8", op="attend", rows=48, longest=5000, hq=14, hkv=2, d=64, page=16, f8=True, heads_first=False),
        # the large model's batch over an 8-bit cache
        dict(name="attend 200 x 4096 f8", op="attend", rows=200, longest=4096, hq=28, hkv=4, d=128, page=32, f8=True, heads_first=False),
        # one conversation's next token, the usual chat settings
        dict(name="sample 1 x 152064", op="sample", rows=1, n=152064, f32=False, k=20, p=0.8, m=0.0, mixed=False),
        # a serving batch, every row with settings of its own, greedy rows among them
        dict(name="sample 64 x 152064", op="sample", rows=64, n=152064, f32=False, k=50, p=0.95, m=0.02, mixed=True),
        # many samples of one prompt from 32-bit logits, nucleus only
        dict(name="sample 256 x 151936 f32", op="sample", rows=256, n=151936, f32=True, k=0, p=0.95, m=0.0, mixed=False),
    ]


HEADS = ((28, 4, 128), (14, 2, 64), (14, 2, 128), (16, 16, 64), (32, 8, 128), (24, 1, 128), (9, 3, 64))


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "sample"))
    if op == "sample":
        n = _spread(rng, 300, 160000)
        rows = _spread(rng, 1, max(1, min(256, 30000000 // n)))
        return dict(op=op, rows=rows, n=n, f32=rng.random() < 0.4, k=rng.choice((0, 1, _spread(rng, 2, n))),
                    p=rng.choice((1.0, round(rng.uniform(0.05, 0.99), 3))), m=rng.choice((0.0, round(rng.uniform(0.001, 0.3), 3))),
                    mixed=rng.random() < 0.5)
    hq, hkv, d = rng.choice(HEADS)
    case = dict(op=op, hq=hq, hkv=hkv, d=d, page=rng.choice((8, 16, 32, 64, 128)), f8=rng.random() < 0.4, heads_first=rng.random() < 0.5)
    if op == "append":
        rows = _spread(rng, 1, 24000)
        return dict(case, rows=rows, seqs=min(rows, _spread(rng, 1, 64)))
    longest = _spread(rng, 1, 100000)
    return dict(case, rows=_spread(rng, 1, max(1, min(200, 250000000 // (longest * hkv * d * 2)))), longest=longest)


def _lengths(case):
    """Keys of each row of an attention case: the first has them all, the others spread below; one free slot in a batch."""
    rng = random.Random("lengths %d %d" % (case["rows"], case["longest"]))
    lens = [case["longest"]] + [rng.randint(1 + case["longest"] // 8, case["longest"]) for _ in range(case["rows"] - 1)]
    if case["rows"] > 8:
        lens[5] = 0
    return lens


def _padding(case):
    """Rows of an append case that are padding: the last eighth of a step's batch."""
    return case["rows"] // 8 if case["rows"] == case["seqs"] and case["rows"] >= 16 else 0


def _prompts(case):
    """(first position, rows) of each sequence of an append case: one row each for a step, ragged prompts otherwise."""
    rows, seqs = case["rows"] - _padding(case), case["seqs"] - _padding(case)
    rng = random.Random("prompts %d %d" % (rows, seqs))
    cuts = sorted(rng.sample(range(1, rows), seqs - 1)) if seqs > 1 else []
    counts = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    return [(rng.randint(0, 2000) if i % 2 or rows == seqs else 0, n) for i, n in enumerate(counts)]


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["n"] * (4 if case["f32"] else 2) + 28), "flops": case["rows"] * case["n"] * 4}
    hq, hkv, d, item = case["hq"], case["hkv"], case["d"], 1 if case["f8"] else 2
    if case["op"] == "append":
        live = case["rows"] - _padding(case)
        # projected rows read, rotation rows read, queries and cache entries written, slots read
        return {"bytes": live * ((hq + 2 * hkv) * d * 2 + 4 * d + hq * d * 2 + 2 * hkv * d * item + 8), "flops": live * (hq + hkv) * d * 8}
    keys = sum(_lengths(case))
    return {"bytes": keys * hkv * d * 2 * item + 2 * case["rows"] * hq * d * 2, "flops": 4 * keys * hq * d}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _pool(pages, case):
    """Zeroed pages, seen as [pages, slots, kv heads, d] whatever their order in memory."""
    dtype = F8 if case["f8"] else torch.bfloat16
    a, b = (case["hkv"], case["page"]) if case["heads_first"] else (case["page"], case["hkv"])
    t = torch.zeros((pages, a, b, case["d"]), device=DEV, dtype=torch.uint8 if case["f8"] else dtype).view(dtype)
    return t.transpose(1, 2) if case["heads_first"] else t


def _rotation(positions, d):
    f = THETA ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    a = torch.cat((a, a), dim=1)
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


def _scales(case, gen):
    """What one stored unit of an 8-bit cache stands for, per kv head."""
    if not case["f8"]:
        return None, None
    return tuple((0.5 + torch.rand(case["hkv"], device=DEV, generator=gen)) * 0.02 for _ in range(2))


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rng = random.Random(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, device=DEV, generator=gen) * std).to(dtype)

    s = dict(case=case, keep={})
    if case["op"] == "sample":
        rows, n = case["rows"], case["n"]
        x = torch.randn((rows, n), device=DEV, generator=gen) * 2
        at = torch.randint(0, n, (rows, min(64, n)), device=DEV, generator=gen)   # the tokens that the context makes likely
        x.scatter_reduce_(1, at, torch.rand(at.shape, device=DEV, generator=gen) * 20 - 2, "amax")
        s["logits"] = x if case["f32"] else x.to(torch.bfloat16)
        s["u"] = torch.rand(rows, device=DEV, generator=gen)
        mixed = case["mixed"]
        every = lambda v, other: [rng.choice((v, other())) if mixed else v for _ in range(rows)]  # noqa: E731
        dev = lambda v, t: torch.tensor(v, device=DEV, dtype=t)  # noqa: E731
        s["t"] = dev(every(0.7, lambda: rng.choice((0.0, 1.0, rng.uniform(0.3, 1.5)))), torch.float32)
        s["k"] = dev(every(case["k"], lambda: rng.choice((0, 1, rng.randint(1, n)))), torch.int32)
        s["p"] = dev(every(case["p"], lambda: rng.choice((1.0, rng.uniform(0.1, 1.0)))), torch.float32)
        s["m"] = dev(every(case["m"], lambda: rng.choice((0.0, rng.uniform(0.0, 0.2)))), torch.float32)
        return s
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    if case["op"] == "append":
        # every sequence has pages of its own, handed out in no order; page 0 is nobody's
        prompts = _prompts(case)
        need = [-(-n // page) + 1 for _, n in prompts]
        ids = list(range(1, 1 + sum(need)))
        rng.shuffle(ids)
        slots, positions = [], []
        for (first, n), c in zip(prompts, need):
            mine = [ids.pop() for _ in range(c)]
            at = first % page
            slots += [mine[(at + i) // page] * page + (at + i) % page for i in range(n)]
            positions += range(first, first + n)
        slots += [-1] * _padding(case)
        positions += [0] * _padding(case)
        s["k_pages"], s["v_pages"] = _pool(1 + sum(need), case), _pool(1 + sum(need), case)
        s["k_scale"], s["v_scale"] = _scales(case, gen)
        s["qkv"] = normal(case["rows"], (hq + 2 * hkv) * d, std=1.5)
        s["q_norm"], s["k_norm"] = 1 + normal(d, std=0.1), 1 + normal(d, std=0.1)
        s["cos"], s["sin"] = _rotation(max(positions) + 1, d)
        s["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
        s["positions"] = torch.tensor(positions, dtype=torch.int32, device=DEV)
        s["q"] = torch.zeros((case["rows"], hq, d), device=DEV, dtype=torch.bfloat16)
        return s
    lens = _lengths(case)
    most = -(-max(lens) // page)
    need = [-(-n // page) for n in lens]
    ids = list(range(1, 1 + sum(need)))
    rng.shuffle(ids)
    table = torch.zeros((case["rows"], most), dtype=torch.int32)
    at = 0
    for r, c in enumerate(need):
        table[r, :c] = torch.tensor(ids[at:at + c], dtype=torch.int32)
        at += c
    s["k_pages"], s["v_pages"] = _pool(1 + sum(need), case), _pool(1 + sum(need), case)
    s["k_scale"], s["v_scale"] = _scales(case, gen)
    for pool, scale in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])):
        for a in range(0, pool.shape[0], 1024):
            x = normal(*pool[a:a + 1024].shape, dtype=torch.float32)
            pool[a:a + 1024] = (x if scale is None else (x / scale[:, None]).clamp(-F8_MAX, F8_MAX)).to(pool.dtype)
    s["q"] = normal(case["rows"], hq, d, std=2.0)
    s["table"], s["lens"] = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["o"] = torch.zeros((case["rows"], hq, d), device=DEV, dtype=torch.bfloat16)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _cache(s):
    """The handle on the pages that a serving program keeps."""
    from bagel_amd import _lib as K
    if "cache" not in s["keep"]:
        s["keep"]["cache"] = K.PagedCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    return K, s["keep"]["cache"]


def _workspace(s, size):
    """Scratch that a serving program keeps, cleared when it is made."""
    if "workspace" not in s["keep"]:
        s["keep"]["workspace"] = torch.zeros(size(), device=DEV, dtype=torch.uint8)
    return s["keep"]["workspace"]


def _own_append(s):
    K, cache = _cache(s)
    K.paged_kv_append(s["qkv"], s["case"]["hq"], cache, s["slots"], Q=s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"], cos_t=s["cos"],
                      sin_t=s["sin"], row_cs=s["positions"], eps=EPS)
    return s["q"], s["k_pages"], s["v_pages"]


def _own_attend(s):
    K, cache = _cache(s)
    c = s["case"]
    ws = _workspace(s, lambda: K.paged_decode_attention_workspace_bytes(c["rows"], c["hq"], c["hkv"], c["d"], c["longest"]))
    K.paged_decode_attention(s["q"], cache, s["table"], s["lens"], s["o"], ws, max_kv_len=c["longest"])
    return s["o"]


def _own_sample(s):
    from bagel_amd import _lib as K
    x = s["logits"]
    ws = _workspace(s, lambda: K.sample_rows_workspace_bytes(x.shape[0], x.shape[1]))
    tokens = torch.empty(x.shape[0], device=DEV, dtype=torch.int32)
    logprobs = torch.empty(x.shape[0], device=DEV, dtype=torch.float32)
    K.sample_rows(x, s["u"], tokens, ws, temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"], logprobs=logprobs)
    return tokens, logprobs


def _plain_append(s):
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    x = s["qkv"].float().view(c["rows"], hq + 2 * hkv, d)
    cos, sin = s["cos"][s["positions"]].float()[:, None], s["sin"][s["positions"]].float()[:, None]

    def rotated(x, weight):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        return x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin

    live = s["slots"] >= 0
    at = s["slots"].clamp(min=0)          # padding lands in slot 0 of page 0, which is nobody's, with what is there
    at, off = torch.div(at, page, rounding_mode="floor").long(), (at % page).long()

    def put(pool, x, scale):
        if scale is not None:
            x = (x / scale[:, None]).clamp(-F8_MAX, F8_MAX)
        byte = torch.uint8 if scale is not None else pool.dtype
        pool.view(byte)[at, off] = torch.where(live[:, None, None], x.to(pool.dtype).view(byte), pool.view(byte)[at, off])

    put(s["k_pages"], rotated(x[:, hq:hq + hkv], s["k_norm"]), s["k_scale"])
    put(s["v_pages"], x[:, hq + hkv:], s["v_scale"])
    s["q"].copy_(torch.where(live[:, None, None], rotated(x[:, :hq], s["q_norm"]).to(torch.bfloat16), s["q"]))
    return s["q"], s["k_pages"], s["v_pages"]


def _plain_attend(s):
    c = s["case"]
    rows, hq, hkv, d = c["rows"], c["hq"], c["hkv"], c["d"]

    def gathered(pool, scale):
        x = pool[s["table"].long()] if not c["f8"] else pool.view(torch.uint8)[s["table"].long()].view(F8)
        x = x.reshape(rows, -1, hkv, d).float()
        return (x if scale is None else x * scale[:, None]).transpose(1, 2).contiguous()      # [rows, kv heads, keys, d]

    k, v = gathered(s["k_pages"], s["k_scale"]), gathered(s["v_pages"], s["v_scale"])
    dead = (torch.arange(k.shape[2], device=DEV) >= s["lens"][:, None])[:, None, None]
    q = s["q"].float().view(rows, hkv, hq // hkv, d)
    x = (torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)).masked_fill(dead, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(x - top)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)   # a free slot gives zeros
    return o.view(rows, hq, d).to(torch.bfloat16)


def _plain_sample(s):
    x, n = s["logits"].double(), s["logits"].shape[1]
    t, k, p, m = s["t"].double()[:, None], s["k"].long()[:, None], s["p"].double()[:, None], s["m"].double()[:, None]
    x, index = torch.sort(x, dim=-1, descending=True, stable=True)                # ties: the lowest index first
    rank = torch.arange(n, device=DEV)
    greedy = t <= 0
    z = (x - x[:, :1]) / torch.where(greedy, 1.0, t)
    w = torch.exp(z)
    kept = torch.where(greedy, 1, torch.where(k <= 0, n, k))
    w = torch.where(rank < kept, w, 0.0)
    sums = torch.cumsum(w, -1)
    w = torch.where((p >= 1) | (sums - w < p * sums[:, -1:]) | (rank == 0), w, 0.0)
    w = torch.where((w >= m) | (rank == 0), w, 0.0)
    sums = torch.cumsum(w, -1)
    total = sums[:, -1:]
    at = (sums <= s["u"].double()[:, None] * total).sum(-1, keepdim=True).clamp(max=n - 1)
    return index.gather(1, at)[:, 0].int(), (z.gather(1, at) - torch.log(total))[:, 0].float()


_plain = {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}
_own = {"append": _own_append, "attend": _own_attend, "sample": _own_sample}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s, case)


def _exact_append(s, case):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    q = torch.zeros((case["rows"], hq, d), dtype=torch.float64, device=DEV)
    shape = (s["k_pages"].shape[0] * page, hkv, d)
    pools = [torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(2)]
    rows = torch.nonzero(s["slots"] >= 0)[:, 0]
    slots = s["slots"][rows].long()
    heads = s["qkv"][rows].double().unflatten(1, (hq + 2 * hkv, d))
    cos, sin = (s[name][s["positions"][rows].long()].double()[:, None, :d // 2] for name in ("cos", "sin"))
    for h in range(hq + hkv):
        x = heads[:, h:h + 1]
        x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * (s["q_norm"] if h < hq else s["k_norm"]).double()
        a, b = x[..., :d // 2], x[..., d // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        if h < hq:
            q[rows, h] = y[:, 0]
        else:
            pools[0][slots, h - hq] = y[:, 0]
    pools[1][slots] = heads[:, hq + hkv:]
    for i, scale in enumerate((s["k_scale"], s["v_scale"])):
        if scale is not None:
            pools[i] = torch.clip(pools[i] / scale.double().view(1, -1, 1), -F8_MAX, F8_MAX)
    return q, pools[0].view(-1, page, hkv, d), pools[1].view(-1, page, hkv, d)


def _exact_attend(s, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    o = torch.zeros((case["rows"], hq, d), dtype=torch.float64, device=DEV)
    for r, n in enumerate(s["lens"].tolist()):
        if n:
            pages = s["table"][r, :-(-n // case["page"])].long()
            k, v = (s[name].view(torch.uint8)[pages].view(F8) if case["f8"] else s[name][pages] for name in ("k_pages", "v_pages"))
            k, v = k.flatten(0, 1)[:n].double(), v.flatten(0, 1)[:n].double()
            for g in range(hkv):
                a, b = k[:, g], v[:, g]
                if case["f8"]:
                    a, b = a * s["k_scale"][g].double(), b * s["v_scale"][g].double()
                mine = slice(g * (hq // hkv), (g + 1) * (hq // hkv))
                o[r, mine] = torch.softmax(s["q"][r, mine].double() @ a.t() * d ** -0.5, dim=1) @ b
    return o


def _exact_sample(s, case):
    import numpy as np
    x = s["logits"].double().cpu().numpy()
    u, t, k, p, m = (s[name].double().cpu().numpy() for name in ("u", "t", "k", "p", "m"))
    tokens, logprobs = [], []
    for r in range(case["rows"]):
        order = np.lexsort((np.arange(case["n"]), -x[r]))
        if t[r] <= 0:
            tokens.append(order[0])
            logprobs.append(0.0)
            continue
        z = (x[r][order] - x[r][order[0]]) / t[r]
        if k[r] >= 1:
            z = z[:int(k[r])]
        w = np.exp(z)
        if p[r] < 1:
            below = np.cumsum(w)
            w = w[:1 + int(np.searchsorted(below, p[r] * below[-1], side="left"))]
        w = w[:max(1, int(np.sum(w >= m[r])))]
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u[r] * sums[-1], side="right")), len(w) - 1)
        tokens.append(order[at])
        logprobs.append(z[at] - np.log(sums[-1]))
    return np.asarray(tokens, dtype=np.int32), np.asarray(logprobs)
