"""Bagel.generate_text with the sampling kernel: filters and given random numbers."""
import pytest
import torch

from tests.scenarios import NEW_TOKEN_IDS, TEXT_CASES
from tests.test_gpu_sample import _want
from tests.test_gpu_text import _context, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["text_tiny_b1", "text_tiny_b2"])
def test_generate_text_with_filters(name):
    """Every sampled token is the definition's for that step's logits; the same numbers give the same text."""
    tc = TEXT_CASES[name]
    model = _model(tc)
    past, kvlens, ropes = _context(model, tc)
    gi = model.prepare_start_tokens(kvlens, ropes, NEW_TOKEN_IDS)
    B, steps = len(kvlens), 12
    u = torch.rand((steps, B), generator=torch.Generator().manual_seed(3))
    for settings in (dict(top_k=20, top_p=0.8, temperature=0.7), dict(min_p=0.05, temperature=1.3), dict(temperature=1.0), dict(top_k=10 ** 9)):
        trace = []
        got = model.generate_text(past_key_values=past, max_length=steps, do_sample=True, uniforms=u, logits_trace=trace, **settings, **gi)
        assert got.shape == (steps, B) and got.dtype == torch.long
        full = lambda v: torch.full((B,), float(v), device="cuda:0")  # noqa: E731
        for t in range(steps - 1):
            want, _ = _want(trace[t], u[t].to("cuda:0"), full(settings.get("temperature", 1.0)), full(min(settings.get("top_k", 0), 1 << 30)),
                            full(settings.get("top_p", 1.0)), full(settings.get("min_p", 0.0)))
            assert torch.equal(got[t + 1], want), (settings, t)
        assert torch.equal(got, model.generate_text(past_key_values=past, max_length=steps, do_sample=True, uniforms=u, **settings, **gi))
    one = model.generate_text(past_key_values=past, max_length=steps, do_sample=True, top_k=1, **gi)
    assert torch.equal(one, model.generate_text(past_key_values=past, max_length=steps, do_sample=False, **gi))


def test_generate_text_refuses_settings_it_cannot_follow():
    tc = TEXT_CASES["text_tiny_b1"]
    model = _model(tc)
    past, kvlens, ropes = _context(model, tc)
    gi = model.prepare_start_tokens(kvlens, ropes, NEW_TOKEN_IDS)
    for bad in (dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=-0.1), dict(top_p=float("nan")), dict(uniforms=torch.rand(3, 1)),
                dict(uniforms=torch.rand(4, 2))):
        with pytest.raises(ValueError):
            model.generate_text(past_key_values=past, max_length=4, do_sample=True, **bad, **gi)
    with pytest.raises(ValueError):
        model.generate_text(past_key_values=past, max_length=4, uniforms=torch.rand(4, 1), **gi)


def test_questions_take_the_filters():
    """interleave_inference hands the sampling settings to the text it decodes."""
    from bagel_amd.inferencer import InterleaveInferencer
    from tests.test_gpu_text import _Tok
    tc = TEXT_CASES["text_tiny_b1"]

    class Tok(_Tok):
        def decode(self, ids):
            return "<|im_start|>" + " ".join(str(int(i)) for i in ids[1:]) + "<|im_end|>"

    inf = InterleaveInferencer(_model(tc), None, Tok(), None, None, NEW_TOKEN_IDS)
    prompt = " ".join(map(str, tc.prompts()[0]))
    ctx = inf.update_context_text(prompt, inf.init_gen_context())
    u = torch.rand((12, 1), generator=torch.Generator().manual_seed(5))
    texts = []
    for settings in (dict(top_k=20, top_p=0.8, uniforms=u), dict(min_p=0.05, uniforms=u), dict(uniforms=u), dict(top_k=1)):
        want = inf.gen_text(ctx, max_length=12, do_sample=True, temperature=1.3, **settings)
        assert inf.interleave_inference([prompt], understanding_output=True, do_sample=True, text_temperature=1.3, max_think_token_n=12,
                                        **settings) == [want]
        assert inf(text=prompt, understanding_output=True, do_sample=True, text_temperature=1.3, max_think_token_n=12, **settings)["text"] == want
        texts.append(want)
    assert texts[3] == inf.interleave_inference([prompt], understanding_output=True, do_sample=False, max_think_token_n=12)[0] != texts[2]
