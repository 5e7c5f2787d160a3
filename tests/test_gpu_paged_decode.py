"""A serving loop on the paged operators: prompts of several requests copied into pages, then steps of append, attention
and sampling through every layer, against the contiguous decode loop fed the same tokens."""
import pytest
import torch

from bagel_amd.config import BagelDims, tiny_dims
from tests.helpers import metrics
from tests.scenarios import NEW_TOKEN_IDS, TextCase
from tests.test_gpu_sample import _want
from tests.test_gpu_text import _context, _logit_bound, _model, _split_ctx

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = torch.bfloat16


class PagedLoop:
    """Pages for every layer, one page table for all of them, handed out as sequences grow."""

    def __init__(self, model, B, page, pages):
        from bagel_amd import _lib as K
        self.K, self.eng, self.B, self.page = K, model.engine, B, page
        d = self.eng.dims
        pool = lambda: torch.zeros((pages, page, d.num_kv_heads, d.head_dim), device=DEV, dtype=BF16)  # noqa: E731
        self.caches = [K.PagedCache(pool(), pool()) for _ in range(d.num_layers)]
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
        self.width = 40
        self.table = torch.zeros((B, self.width), dtype=torch.int32)
        self.owned = [0] * B
        self.lens = [0] * B
        self.ws = torch.zeros(K.paged_decode_attention_workspace_bytes(B, d.num_heads, d.num_kv_heads, d.head_dim, self.width * page), device=DEV,
                              dtype=torch.uint8)

    def slots(self, b, n):
        """Slots of the sequence's next n tokens."""
        out = []
        for i in range(self.lens[b], self.lens[b] + n):
            if i // self.page >= self.owned[b]:
                self.table[b, self.owned[b]] = self.free.pop()
                self.owned[b] += 1
            out.append(int(self.table[b, i // self.page]) * self.page + i % self.page)
        self.lens[b] += n
        return out

    def finish(self, b):
        self.free += self.table[b, :self.owned[b]].tolist()
        self.owned[b] = self.lens[b] = 0

    def adopt(self, b, keys, values):
        """Copies a context ([n, kv heads, head_dim] per layer, already rotated) into pages."""
        n = keys[0].shape[0]
        slots = torch.tensor(self.slots(b, n), dtype=torch.int32, device=DEV)
        for cache, k, v in zip(self.caches, keys, values):
            self.K.paged_kv_append(torch.cat((k.flatten(1), v.flatten(1)), 1), 0, cache, slots)

    def step(self, tokens, positions, live):
        """Logits of one new token per live sequence."""
        K, d, w = self.K, self.eng.dims, self.eng.w
        from bagel_amd.engine import rope_table
        B, H, D = self.B, d.hidden_size, d.head_dim
        qkv_dim = d.q_dim + 2 * d.kv_dim
        slots = torch.tensor([self.slots(b, 1)[0] if live[b] else -1 for b in range(B)], dtype=torch.int32, device=DEV)
        lens = torch.tensor([self.lens[b] if live[b] else 0 for b in range(B)], dtype=torch.int32, device=DEV)
        table = self.table.to(DEV)
        cos, sin = rope_table(positions, D, d.rope_theta, DEV)
        cs = torch.arange(B, dtype=torch.int32, device=DEV)
        new = lambda *s: torch.zeros(s, device=DEV, dtype=BF16)  # noqa: E731
        X, Xn, QKV, Q, O, Hm = new(B, H), new(B, H), new(B, qkv_dim), new(B, d.num_heads, D), new(B, d.num_heads, D), new(B, d.intermediate_size)
        logits = new(B, w.lm_head.shape[0])
        skw = torch.empty(16 * B * max(2 * d.intermediate_size, qkv_dim, logits.shape[1]), device=DEV)
        K.gather_rows(w.embed_tokens, tokens, X, B)
        for lw, cache in zip(w.layers, self.caches):
            K.rmsnorm(X, Xn, lw.ln_in[1], None, B, d.rms_norm_eps)
            K.skinny_gemm(Xn, lw.wqkv[1], QKV, skw, bias=lw.bqkv[1])
            K.paged_kv_append(QKV, d.num_heads, cache, slots, Q=Q, q_norm=lw.qn[1], k_norm=lw.kn[1], cos_t=cos, sin_t=sin, row_cs=cs,
                              eps=d.rms_norm_eps, und_rounding=True)
            K.paged_decode_attention(Q, cache, table, lens, O, self.ws, max_kv_len=max(self.lens))
            K.skinny_gemm(O.flatten(1), lw.wo[1], X, skw, residual=X, epilogue=K.SK_RESIDUAL)
            K.rmsnorm(X, Xn, lw.ln_post[1], None, B, d.rms_norm_eps)
            K.skinny_gemm(Xn, lw.wgu[1], Hm, skw, epilogue=K.SK_SWIGLU)
            K.skinny_gemm(Hm, lw.wd[1], X, skw, residual=X, epilogue=K.SK_RESIDUAL)
        K.rmsnorm(X, Xn, w.norm[1], None, B, d.rms_norm_eps)
        K.skinny_gemm(Xn, w.lm_head, logits, skw)
        return logits


WIDE = BagelDims(hidden_size=896, intermediate_size=512, num_layers=2, num_heads=14, num_kv_heads=2, vocab_size=512)


@pytest.mark.parametrize("dims,page", [(tiny_dims(3), 8), (tiny_dims(2), 64), (WIDE, 16)])
def test_paged_decoding_equals_the_contiguous_loop(dims, page):
    from bagel_amd import _lib as K
    steps = 10
    tc = TextCase("paged", dims, [3, 62, 140, 65], steps, weight_seed=2)
    model = _model(tc)
    past, kvlens, ropes = _context(model, tc)
    gi = model.prepare_start_tokens(kvlens, ropes, NEW_TOKEN_IDS)
    ctx_k, ctx_v = _split_ctx(model, past, kvlens)
    B, n = len(kvlens), dims.vocab_size
    loop = PagedLoop(model, B, page, 120)
    for b in range(B):
        loop.adopt(b, ctx_k[b], ctx_v[b])
    gen = torch.Generator(device=DEV).manual_seed(4)
    settings = dict(t=torch.full((B,), 0.9, device=DEV), k=torch.full((B,), 50, device=DEV, dtype=torch.int32), p=torch.full((B,), 0.9, device=DEV),
                    m=torch.full((B,), 0.01, device=DEV))
    sample_ws = torch.empty(K.sample_rows_workspace_bytes(B, n), device=DEV, dtype=torch.uint8)
    tokens = torch.tensor(gi["packed_start_tokens"].tolist(), dtype=torch.int32, device=DEV)
    pos0 = gi["packed_query_position_ids"].tolist()
    fed, trace = [tokens.clone()], []
    live = [True] * B
    for t in range(steps):
        if t == 6:                       # one request ends: its pages go back, its row becomes padding
            live[1] = False
            loop.finish(1)
        logits = loop.step(tokens, [p + t for p in pos0], live)
        trace.append(logits.float().cpu())
        u = torch.rand(B, device=DEV, generator=gen)
        nxt = torch.empty_like(tokens)
        K.sample_rows(logits, u, nxt, sample_ws, temperature=settings["t"], top_k=settings["k"], top_p=settings["p"], min_p=settings["m"])
        assert torch.equal(nxt.long(), _want(logits, u, **settings)[0])
        tokens = nxt
        fed.append(tokens.clone())
    want, at = [], [0]

    def forced(_):
        at[0] += 1
        return fed[at[0]].long()

    model.engine.decode_tokens(gi["packed_start_tokens"].tolist(), pos0, kvlens, ctx_k, ctx_v, steps, sample_fn=forced, logits_trace=want)
    for t in range(steps):
        rows = [b for b in range(B) if b != 1 or t < 6]
        ref = want[t].float().cpu()[rows]
        ma, cos = metrics(trace[t][rows], ref)
        # the bound that the contiguous loop's own logits are held to against another order of the same sums
        assert ma <= _logit_bound(ref) and cos >= 0.9999, (t, ma, cos)
