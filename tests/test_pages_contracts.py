"""Calls of the paged FP8 cache's entry points that are refused, and their 64-bit oracle against
independent conversions (no GPU)."""
import numpy as np
import pytest
import torch

import pages_ref
import w4amd

A = 64  # an address that no check may touch


def _view(c, H=2, D=64, page=16, npages=8, q_k=A, s_k=A, q_v=A, s_v=A):
    return c.f8_pages_view(H, D, page, npages, q_k, s_k, q_v, s_v)


def _batch(c, nseq=3, tokens=3, max_q=1, max_len=100, bt=A, stride=8, lens=A, cu=A):
    return c.paged_batch(nseq, tokens, max_q, max_len, bt, stride, lens, cu)


def test_tables_refuse_what_they_cannot_do():
    c = w4amd.capi()
    good = dict(page=16, npages=8, cached=128, added=192, free_pages=A, free_range=A, slots=A, positions=A, result=A)

    def refused(text, batch=None, **change):
        with pytest.raises(ValueError, match=text):
            c.paged_tables(batch if batch is not None else _batch(c), **{**good, **change})

    refused("bad dims", _batch(c, nseq=0))
    refused("bad dims", _batch(c, tokens=-1))
    refused("bad dims", _batch(c, stride=0))
    refused("page geometry", page=0)
    refused("page geometry", npages=0)
    refused("page geometry", page=1 << 16, npages=1 << 15)
    for name in ("cached", "added", "free_pages", "free_range", "result"):
        refused("null pointer", **{name: 0})
    for name in ("bt", "lens", "cu"):
        refused("null pointer", _batch(c, **{name: 0}))
    refused("null slots", slots=0)
    refused("null slots", positions=0)
    refused("lens is an output", cached=A)
    refused("lens is an output", added=A)


def _views_refused(call, c):
    for change, text in (({"H": 0}, "bad dims"), ({"D": 0}, "bad dims"), ({"D": 516}, "512"), ({"D": 66}, "multiple of 4"),
                         ({"page": 0}, "page geometry"), ({"npages": 0}, "page geometry"),
                         ({"page": 1 << 20, "npages": 1 << 11}, "page geometry"), ({"H": 65536}, "too many heads"),
                         ({"q_k": 0}, "null pointer"), ({"s_k": 0}, "null pointer"), ({"q_v": 0}, "null pointer"),
                         ({"s_v": 0}, "null pointer"), ({"q_k": A + 2}, "4-byte aligned"), ({"q_v": A + 1}, "4-byte aligned")):
        with pytest.raises(ValueError, match=text):
            call(_view(c, **change))


def test_append_refuses_what_it_cannot_do():
    c = w4amd.capi()
    _views_refused(lambda v: c.quantize_f8_pages(v, A, A, 0, A, 3, A), c)
    for args, text in (((0, A, 0, A, 3, A), "null io"), ((A, 0, 0, A, 3, A), "null io"), ((A, A, 0, 0, 3, A), "null io"),
                       ((A, A, 0, A, 3, 0), "null io"), ((A, A, 127, A, 3, A), "row_stride"), ((A, A, -1, A, 3, A), "row_stride"),
                       ((A, A, 0, A, -1, A), "bad dims"), ((A, A, 0, A, 1 << 29, A), "too many rows")):
        with pytest.raises(ValueError, match=text):
            c.quantize_f8_pages(_view(c), *args)
    c.quantize_f8_pages(_view(c), A, A, 0, 0, 0, A)  # no tokens: nothing is launched


def test_attention_refuses_what_it_cannot_do():
    c = w4amd.capi()
    _views_refused(lambda v: c.attention_f8_pages(v, _batch(c), 2, 1, A, 0, A, A, 1 << 30), c)
    _views_refused(lambda v: c.attention_f8_pages_workspace(v, _batch(c), 2), c)

    def refused(text, batch=None, group=2, causal=1, q=A, q_stride=0, out=A, space=A, space_bytes=1 << 30):
        with pytest.raises(ValueError, match=text):
            c.attention_f8_pages(_view(c), batch if batch is not None else _batch(c), group, causal, q, q_stride, out, space,
                                 space_bytes)

    for change in ({"nseq": 0}, {"tokens": -1}, {"max_q": 0}, {"max_len": 0}, {"stride": 0}):
        refused("bad dims", _batch(c, **change))
    refused("null pointer", _batch(c, bt=0))
    refused("null pointer", _batch(c, lens=0))
    refused("need cu_q", _batch(c, cu=0, max_q=2))
    refused("need cu_q", _batch(c, cu=0, tokens=4))
    refused("query group", group=0)
    refused("query group", group=65)
    refused("too many rows", _batch(c, nseq=1 << 30, tokens=3))
    refused("too many rows", _batch(c, tokens=1 << 30))
    refused("null io", q=0)
    refused("null io", out=0)
    refused("causal", causal=2)
    refused("q_stride", q_stride=255)
    long = _batch(c, nseq=1, tokens=1, max_len=100000, stride=10000)
    need = c.attention_f8_pages_workspace(_view(c), long, 2)
    assert need > 0
    refused("workspace too small", long, space_bytes=need - 1)
    refused("workspace too small", long, space=0, space_bytes=need)
    refused("16-byte aligned", long, space=A + 8, space_bytes=need)


def test_encoder_agrees_with_another():
    """Every half, over several scales, against torch's conversion; the tie rule on every border."""
    x = np.arange(1 << 16, dtype=np.uint16).view(np.float16)
    x = x[np.isfinite(x)].astype(np.float64)
    for scale in (1.0, 0.015, 2.0 ** -20, 3.7):
        y = (x / scale).astype(np.float32)
        want = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        assert np.array_equal(pages_ref.encode(y), want)
    mids = pages_ref._MIDS
    codes = pages_ref.encode(mids)
    assert (codes % 2 == 0).all() and (np.abs(pages_ref.VALUES[codes] - mids) == (mids - pages_ref._MAGS[:-1])).all()


def test_scale_never_saturates():
    x = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)
    for a in x[::97]:
        s = pages_ref.scale_for(a)
        assert float(s) * 448 >= a and (s == 0 or float(np.nextafter(s, np.float16(0))) * 448 < a)
