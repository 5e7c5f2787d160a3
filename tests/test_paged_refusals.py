"""What the paged cache's entry points refuse, on the host: nothing here reaches a device."""
import ctypes

import pytest
import torch

from bagel_amd import _lib as K

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn


def _pools(pages=4, page=16, heads=2, d=64, dtype=BF16):
    raw = torch.uint8 if dtype == F8 else torch.int16
    return tuple(torch.zeros((pages, page, heads, d), dtype=raw).view(dtype) for _ in range(2))


def _scale(heads=2):
    return torch.ones(heads)


@pytest.mark.parametrize("make,message", [
    (lambda: K.PagedCache(_pools()[0][0], _pools()[1][0]), "two pools"),
    (lambda: K.PagedCache(_pools()[0], _pools(pages=5)[0]), "two pools"),
    (lambda: K.PagedCache(*_pools(pages=0)), "two pools"),
    (lambda: K.PagedCache(_pools()[0].float(), _pools()[1].float()), "bfloat16 or float8"),
    (lambda: K.PagedCache(_pools()[0], _pools(dtype=F8)[0]), "bfloat16 or float8"),
    (lambda: K.PagedCache(*(t.transpose(2, 3) for t in _pools())), "must be contiguous"),
    (lambda: K.PagedCache(*_pools(dtype=F8)), "k_scale and v_scale"),
    (lambda: K.PagedCache(*_pools(dtype=F8), k_scale=_scale()), "k_scale and v_scale"),
    (lambda: K.PagedCache(*_pools(), k_scale=_scale(), v_scale=_scale()), "k_scale and v_scale"),
    (lambda: K.PagedCache(*_pools(dtype=F8), k_scale=_scale(3), v_scale=_scale(3)), "scales are"),
    (lambda: K.PagedCache(*_pools(dtype=F8), k_scale=_scale().double(), v_scale=_scale().double()), "scales are")])
def test_cache_refusals(make, message):
    with pytest.raises(RuntimeError, match=message):
        make()


def _append(**change):
    a = dict(qkv=torch.zeros((3, (4 + 2 * 2) * 64), dtype=BF16), Hq=4, cache=K.PagedCache(*_pools()),
             row_slot=torch.zeros(3, dtype=torch.int32), Q=torch.zeros((3, 4, 64), dtype=BF16))
    a.update(change)
    return K.paged_kv_append(**a)


@pytest.mark.parametrize("change,message", [
    (dict(Hq=3), "qkv"), (dict(Hq=0), "without query heads"), (dict(Hq=-1), "without query heads"),
    (dict(qkv=torch.zeros((3, 512))), "qkv"), (dict(qkv=torch.zeros((512, 3), dtype=BF16).t()), "contiguous"),
    (dict(row_slot=torch.zeros(3, dtype=torch.int64)), "row_slot"), (dict(row_slot=torch.zeros(4, dtype=torch.int32)), "row_slot"),
    (dict(row_slot=torch.zeros(6, dtype=torch.int32)[::2]), "row_slot"),
    (dict(Q=torch.zeros((2, 4, 64), dtype=BF16)), "rows"), (dict(Q=torch.zeros((3, 5, 64), dtype=BF16)), "Q"),
    (dict(q_norm=torch.ones(64)), "norm weights"), (dict(k_norm=torch.ones(128, dtype=BF16)), "norm weights"),
    (dict(cos_t=torch.ones((9, 64), dtype=BF16)), "come together"),
    (dict(cos_t=torch.ones((9, 64), dtype=BF16), sin_t=torch.ones((9, 64), dtype=BF16)), "come together"),
    (dict(cos_t=torch.ones((9, 64)), sin_t=torch.ones((9, 64)), row_cs=torch.zeros(3, dtype=torch.int32)), "rotation tables"),
    (dict(cos_t=torch.ones((9, 64), dtype=BF16), sin_t=torch.ones((8, 64), dtype=BF16), row_cs=torch.zeros(3, dtype=torch.int32)), "rotation tables"),
    (dict(cos_t=torch.ones((9, 64), dtype=BF16), sin_t=torch.ones((9, 64), dtype=BF16), row_cs=torch.zeros(3, dtype=torch.int64)), "row_cs"),
    (dict(), "device tensor")])
def test_append_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _append(**change)


def _attend(**change):
    a = dict(Q=torch.zeros((3, 4, 64), dtype=BF16), cache=K.PagedCache(*_pools()), page_table=torch.zeros((3, 2), dtype=torch.int32),
             kv_lens=torch.zeros(3, dtype=torch.int32), O=torch.zeros((3, 4, 64), dtype=BF16), workspace=torch.zeros(1 << 16, dtype=torch.uint8))
    a.update(change)
    return K.paged_decode_attention(**a)


@pytest.mark.parametrize("change,message", [
    (dict(Q=torch.zeros((3, 3, 64), dtype=BF16), O=torch.zeros((3, 3, 64), dtype=BF16)), "multiple of 2 heads"),
    (dict(Q=torch.zeros((3, 4, 128), dtype=BF16), O=torch.zeros((3, 4, 128), dtype=BF16)), "multiple of 2 heads"),
    (dict(O=torch.zeros((2, 4, 64), dtype=BF16)), "multiple of 2 heads"), (dict(Q=torch.zeros((3, 4, 64))), "Q"),
    (dict(O=torch.zeros((3, 4, 64))), "O"), (dict(Q=torch.zeros((3, 4, 128), dtype=BF16)[:, :, ::2]), "contiguous"),
    (dict(page_table=torch.zeros((3, 2), dtype=torch.int64)), "page_table"), (dict(page_table=torch.zeros((2, 2), dtype=torch.int32)), "page_table"),
    (dict(page_table=torch.zeros((3, 0), dtype=torch.int32)), "page_table"), (dict(page_table=torch.zeros((2, 3), dtype=torch.int32).t()), "page_table"),
    (dict(kv_lens=torch.zeros(3, dtype=torch.int64)), "kv_lens"), (dict(max_kv_len=-1), "max_kv_len"),
    (dict(softmax_scale=0.0), "softmax_scale"), (dict(softmax_scale=float("nan")), "softmax_scale"),
    (dict(workspace=torch.zeros((2, 1 << 16), dtype=torch.uint8).t()), "workspace"), (dict(), "device tensor")])
def test_attention_refusals(change, message):
    with pytest.raises(RuntimeError, match=message):
        _attend(**change)


# ---- the C entry points: addresses that are never followed ------------------------------------------------------------

A = 1 << 20


def _c_cache(**change):
    a = dict(k=A, v=A, k_page_stride=16 * 2 * 64, k_slot_stride=2 * 64, k_head_stride=64, v_page_stride=16 * 2 * 64, v_slot_stride=2 * 64,
             v_head_stride=64, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, e4m3=0, k_scale=None, v_scale=None)
    a.update(change)
    s = K._PagedCacheStruct()
    for name, value in a.items():
        setattr(s, name, value)
    return s


def _c_append(cache=None, qkv=A, ld=512, rows=3, hq=4, qn=None, kn=None, cos=None, sin=None, n=0, cs=None, slot=A, q=A, ldq=256):
    fn = K._declared("bagel_paged_kv_append_bf16", K.VP, K.L, K.I, K.I, K.VP, K.VP, K.VP, K.VP, K.VP, K.I, K.VP, K.VP, K.VP, K.L, K.F, K.I, K.VP)
    return fn(qkv, ld, rows, hq, ctypes.byref(cache) if cache is not None else None, qn, kn, cos, sin, n, cs, slot, q, ldq, 1e-6, 0, None)


def _c_attend(cache=None, q=A, ldq=256, rows=3, hq=4, table=A, stride=2, width=2, lens=A, bound=0, o=A, ldo=256, ws=A, ws_bytes=1 << 20):
    fn = K._declared("bagel_paged_decode_attention_bf16", K.VP, K.L, K.I, K.I, K.VP, K.VP, K.L, K.I, K.VP, K.L, K.VP, K.L, K.F, K.VP, K.L, K.VP)
    return fn(q, ldq, rows, hq, ctypes.byref(cache) if cache is not None else None, table, stride, width, lens, bound, o, ldo, 0.0, ws, ws_bytes, None)


BAD_CACHES = [
    (dict(k=None), "null cache"), (dict(v=None), "null cache"), (dict(head_dim=96), "head_dim"), (dict(num_kv_heads=0), "kv heads"),
    (dict(num_pages=0), "pages"), (dict(page_size=4), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=0), "page_size"),
    (dict(page_size=-16), "page_size"), (dict(num_pages=1 << 28), "32 bits"), (dict(e4m3=2), "e4m3"), (dict(e4m3=1), "k_scale"),
    (dict(k=A + 2), "16-byte"), (dict(k_slot_stride=132), "16-byte"), (dict(v_head_stride=68), "16-byte"),
    (dict(e4m3=1, k_scale=A, v_scale=A, v_head_stride=72), "16-byte"), (dict(v_slot_stride=32), "below head_dim"), (dict(k_head_stride=0), "below head_dim")]


@pytest.mark.parametrize("change,message", BAD_CACHES)
def test_c_entries_refuse_the_cache(change, message):
    for call in (_c_append, _c_attend):
        assert call(_c_cache(**change)) != 0 and message in K.lib().bagel_last_error().decode()
    assert _c_append(None) != 0 and _c_attend(None) != 0


@pytest.mark.parametrize("change,message", [
    (dict(qkv=None), "null operand"), (dict(slot=None), "null operand"), (dict(rows=-1), "rows"), (dict(hq=-1), "Hq"), (dict(ld=508), "leading dim"),
    (dict(ld=504), "leading dim"), (dict(ldq=248), "of Q"), (dict(cos=A), "rotation"), (dict(cos=A, sin=A, n=4), "rotation"),
    (dict(cos=A, sin=A, cs=A, n=0), "rotation"), (dict(qkv=A + 2), "misaligned"), (dict(q=A + 8), "misaligned"), (dict(kn=A + 2), "misaligned")])
def test_c_append_refusals(change, message):
    assert _c_append(_c_cache(), **change) != 0 and message in K.lib().bagel_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "null operand"), (dict(o=None), "null operand"), (dict(table=None), "null operand"), (dict(lens=None), "null operand"),
    (dict(ws=None), "null operand"), (dict(rows=-1), "rows"), (dict(rows=65536), "rows"), (dict(hq=3), "multiple"), (dict(hq=0), "multiple"),
    (dict(width=0), "page table"), (dict(stride=1), "page table"), (dict(width=1 << 27, stride=1 << 27), "2^30"), (dict(ldq=252), "leading dim"),
    (dict(ldo=248), "leading dim"), (dict(q=A + 2), "misaligned"), (dict(ws=A + 4), "misaligned"), (dict(ws_bytes=64), "workspace of 64 bytes")])
def test_c_attention_refusals(change, message):
    assert _c_attend(_c_cache(), **change) != 0 and message in K.lib().bagel_last_error().decode()


def test_nothing_to_do_is_no_error():
    assert _c_append(_c_cache(), rows=0, qkv=None, slot=None) == 0
    assert _c_attend(_c_cache(), rows=0, q=None, o=None) == 0
    assert K.paged_decode_attention_workspace_bytes(0, 4, 2, 64, 100) == 0


def test_workspace_of_unknown_lengths():
    """A bound of 0 means the same to the workspace's size as to the call: rows of any length."""
    for rows, hq, hkv, d in ((1, 28, 4, 128), (3, 4, 2, 64), (9, 24, 1, 128), (300, 14, 2, 64)):
        sizes = [K.paged_decode_attention_workspace_bytes(rows, hq, hkv, d, n) for n in (1, 600, 9000, 1 << 20, 1 << 30)]
        assert sizes == sorted(sizes) and K.paged_decode_attention_workspace_bytes(rows, hq, hkv, d, 0) == sizes[-1]


@pytest.mark.parametrize("scale", [1e-60, -1e-60, 1e300, -1e300])
def test_attention_refuses_scales_that_32_bits_do_not_hold(scale):
    """The entry point takes 32 bits, where these are 0 (which asks for 1 / sqrt(head_dim) instead) and infinity."""
    with pytest.raises(RuntimeError, match="softmax_scale"):
        _attend(softmax_scale=scale)
