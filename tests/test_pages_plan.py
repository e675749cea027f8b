"""Which kernels a call of paged FP8 attention runs, how it splits positions, and bounds that calls are refused past
(no GPU)."""
import pytest

import w4amd

A = 64  # an address that no check may touch


def plan(H=8, D=128, page=16, npages=100, nseq=1, tokens=1, max_q=1, max_len=1000, stride=1 << 16, group=4, cu=A, q_k=A):
    c = w4amd.capi()
    view = c.f8_pages_view(H, D, page, npages, q_k, A, A, A)
    return c.attention_f8_pages_plan_for(view, c.paged_batch(nseq, tokens, max_q, max_len, A, stride, A, cu), group)


def test_kernels_of_a_call():
    assert plan(nseq=8, tokens=8, max_len=32768)[:2] == (1, 4)                 # a token each
    assert plan(nseq=8, tokens=40, max_q=5, max_len=32768)[:2] == (1, 20)      # a few each
    assert plan(tokens=100, max_q=100, max_len=100)[:2] == (1, 400)            # a small prompt
    assert plan(tokens=4096, max_q=4096, max_len=4096)[:2] == (2, 0)           # a prompt
    assert plan(nseq=16, tokens=527, max_q=512, max_len=8192)[:2] == (4, 16)   # a chunk next to decoding sequences
    assert plan(nseq=16, tokens=527, max_q=512, max_len=8192, page=24)[:2] == (3, 16)
    assert plan(nseq=16, tokens=527, max_q=512, max_len=8192, group=20)[:2] == (3, 32)
    assert plan(nseq=16, tokens=527, max_q=512, max_len=8192, group=40)[:2] == (2, 0)
    for other in (dict(D=80), dict(D=512), dict(q_k=A + 4)):                   # nothing but the vector kernel takes these
        assert plan(nseq=16, tokens=527, max_q=512, max_len=8192, **other)[:2] == (0, 0)


def test_splits_cover_the_longest_sequence():
    for kernel in ({}, {"D": 80}, {"page": 24}):
        for tokens in (1, 40, 128, 512, 1024, 5000):
            for nseq in (1, 2, 16):
                for max_len in (1, 63, 64, 65, 512, 1000, 8192, 100_000, 1_000_000):
                    _, few, length, splits = plan(nseq=nseq, tokens=tokens, max_q=tokens, max_len=max_len, **kernel)
                    case = (kernel, tokens, nseq, max_len)
                    assert splits >= 1 and length >= 1 and (splits - 1) * length < max_len <= splits * length, case


def test_a_plan_refuses_what_the_call_refuses():
    for change, text in (({"D": 516}, "512"), ({"group": 65}, "query group"), ({"max_len": 0}, "bad dims"), ({"cu": 0, "tokens": 2}, "need cu_q")):
        with pytest.raises(ValueError, match=text):
            plan(**change)
    c = w4amd.capi()
    view, batch = c.f8_pages_view(8, 128, 16, 100, A, A, A, A), c.paged_batch(1, 1, 1, 100, A, 100, A, A)
    assert c.load().w4_attention_f8_pages_plan_for(view, batch, 4, None) != 0


def test_bounds_of_positions():
    """max_len counts as far as the tables reach.  Up to 2^30 positions every plan covers them; what is more is refused."""
    for kernel in ({}, {"D": 80}, {"page": 1000}, {"nseq": 2, "tokens": 40}, {"nseq": 2, "tokens": 40, "group": 20}):
        for tokens, max_q in ((2, 1), (40, 30), (1000, 990), (300_000, 300_000)):
            base = {"nseq": 2, "page": 1024, "stride": 1 << 21, "H": 1, **kernel, "tokens": tokens, "max_q": max_q}
            for max_len in (1 << 30, (1 << 30) - 1, (1 << 30) - 127):
                _, _, length, splits = plan(max_len=max_len, **base)
                assert 1 <= length <= max_len + 255 and (splits - 1) * length < max_len <= splits * length, (base, max_len)
            for max_len in ((1 << 30) + 1, 2147483000, 2 ** 31 - 1):
                with pytest.raises(ValueError, match="pass 2.30 positions"):
                    plan(max_len=max_len, **base)
            short = {**base, "stride": 50}
            assert plan(max_len=2 ** 31 - 1, **short) == plan(max_len=50 * short["page"], **short)
    assert plan(max_len=2 ** 31 - 1, page=1024, stride=1 << 20)[3] >= 1   # a table of 2^30 positions


def test_calls_past_the_bounds_of_positions_are_refused():
    c = w4amd.capi()
    view, batch = c.f8_pages_view(1, 128, 1024, 100, A, A, A, A), c.paged_batch(2, 41, 40, 2 ** 31 - 1, A, 1 << 21, A, A)
    with pytest.raises(ValueError, match="pass 2.30 positions"):
        c.attention_f8_pages(view, batch, 4, 1, A, 0, A, A, 1 << 40)
    with pytest.raises(ValueError, match="pass 2.30 positions"):
        c.attention_f8_pages_workspace(view, batch, 4)


def test_one_launch_or_two():
    """Decoding sequences next to a chunk: one launch as long as units of the few-rows kernel are split, over half of the card
    or over all of it."""
    many = dict(tokens=5000, max_q=512, max_len=8192)
    for nseq, H, D, kind in ((2, 8, 128, 4), (255, 8, 128, 4), (256, 8, 128, 4), (256, 15, 64, 4), (256, 16, 64, 3), (257, 1, 128, 3),
                             (255, 8, 256, 4), (256, 8, 256, 3), (255, 16, 96, 4)):
        assert plan(nseq=nseq, H=H, D=D, **many)[:2] == (kind, 16), (nseq, H, D)
    assert plan(nseq=256, H=8, tokens=200_000, max_q=512, max_len=512)[0] == 3  # (up to 512 positions no unit is split)


def test_append_refuses_pages_past_what_it_counts():
    c = w4amd.capi()

    def append(D, page):
        c.quantize_f8_pages(c.f8_pages_view(1, D, page, 1, A, A, A, A), A, A, 0, 0, 0, A)

    append(512, 1 << 23), append(4, 1 << 30), append(128, 1 << 25)
    for D, page in ((512, (1 << 23) + 1), (512, (1 << 31) - 1), (8, (1 << 29) + 1)):
        with pytest.raises(ValueError, match="2.32 bytes"):
            append(D, page)


def test_tables_refuse_sequences_past_what_they_count():
    c = w4amd.capi()
    for nseq in ((1 << 30) + 1, 2 ** 31 - 1000, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="2.30 sequences"):
            c.paged_tables(c.paged_batch(nseq, 3, 1, 100, A, 8, A, A), 16, 8, 128, 192, A, A, A, A, A)
