"""What the sampling entry points refuse, on the host: nothing here reaches a device."""
import pytest
import torch

from bagel_amd import _lib as K


def _sample(**change):
    f = lambda: torch.zeros(3)  # noqa: E731
    a = dict(logits=torch.zeros((3, 10), dtype=torch.bfloat16), uniforms=f(), tokens=torch.zeros(3, dtype=torch.int32),
             workspace=torch.zeros(1 << 17, dtype=torch.uint8), temperature=f(), top_k=torch.zeros(3, dtype=torch.int32), top_p=f(), min_p=f(),
             logprobs=f())
    a.update(change)
    return K.sample_rows(**a)


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros((3, 10), dtype=torch.float16)), "logits"), (dict(logits=torch.zeros(30)), "logits"),
    (dict(logits=torch.zeros((10, 3)).t()), "logits"), (dict(uniforms=torch.zeros(4)), "uniforms"),
    (dict(uniforms=torch.zeros(3, dtype=torch.float64)), "uniforms"), (dict(tokens=torch.zeros(3, dtype=torch.int64)), "tokens"),
    (dict(temperature=torch.zeros((3, 1))), "temperature"), (dict(top_k=torch.zeros(3)), "top_k"), (dict(top_p=torch.zeros(6)[::2]), "top_p"),
    (dict(min_p=torch.zeros(2)), "min_p"), (dict(logprobs=torch.zeros(3, dtype=torch.bfloat16)), "logprobs"),
    (dict(workspace=torch.zeros((2, 1 << 16), dtype=torch.uint8).t()), "workspace"), (dict(), "device tensor")])
def test_sampling_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _sample(**change)


A = 1 << 20


def _c_sample(logits=A, ld=100, rows=3, n=100, f32=0, u=A, t=None, k=None, p=None, m=None, tokens=A, logprobs=None, ws=A, ws_bytes=1 << 20):
    fn = K._declared("bagel_sample_rows", K.VP, K.L, K.I, K.I, K.I, K.VP, K.VP, K.VP, K.VP, K.VP, K.VP, K.VP, K.VP, K.L, K.VP)
    return fn(logits, ld, rows, n, f32, u, t, k, p, m, tokens, logprobs, ws, ws_bytes, None)


@pytest.mark.parametrize("change,message", [
    (dict(logits=None), "null operand"), (dict(u=None), "null operand"), (dict(tokens=None), "null operand"), (dict(ws=None), "null operand"),
    (dict(rows=-1), "rows"), (dict(rows=65536), "rows"), (dict(n=0), "tokens"), (dict(n=(1 << 20) + 1, ld=1 << 21), "tokens"), (dict(ld=99), "leading dim"),
    (dict(f32=2), "logits_f32"), (dict(logits=A + 1), "misaligned"), (dict(logits=A + 2, f32=1), "misaligned"), (dict(ws=A + 8), "misaligned"),
    (dict(ws_bytes=1000), "workspace of 1000 bytes")])
def test_c_sampling_refusals(change, message):
    assert _c_sample(**change) != 0 and message in K.lib().bagel_last_error().decode()


def test_no_rows_is_no_error():
    assert _c_sample(rows=0, logits=None, u=None, tokens=None, ws=None) == 0
    assert K.sample_rows_workspace_bytes(0, 100) == 0 and K.sample_rows_workspace_bytes(5, 0) == 0


def test_workspace_serves_fewer_rows():
    for n in (1000, 32000, 61265, 152064, 1 << 20):
        sizes = [K.sample_rows_workspace_bytes(rows, n) for rows in range(1, 90)]
        assert sizes == sorted(sizes) and sizes[0] > 0
