"""Serving over a paged FP8 cache on the device: pages and slots, the write of new tokens, attention, and
the three as one step, against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import pages_ref
import w4amd
from devutil import DEV, ptr, to_dev

pytestmark = pytest.mark.gpu


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(DEV)


def same(got, want):
    bad = np.argwhere(got != want)
    assert not len(bad), (len(bad), bad[0].tolist(), got[tuple(bad[0])], want[tuple(bad[0])])


# ---- tables ----------------------------------------------------------------------------


def run_tables(bt, page, npages, tokens, cached, added, free_pages, free_range, stream=0):
    c = w4amd.capi()
    nseq, R = bt.shape
    d = [i32(a) for a in (bt, cached, added, free_pages, free_range)]
    lens, cu, result = i32(np.full(nseq, 77)), i32(np.full(nseq + 1, 77)), i32([77, 77])
    slots, positions = i32(np.full(tokens, 77)), i32(np.full(tokens, 77))
    batch = c.paged_batch(nseq, tokens, 1, 1, ptr(d[0]), R, ptr(lens), ptr(cu))
    c.paged_tables(batch, page, npages, ptr(d[1]), ptr(d[2]), ptr(d[3]), ptr(d[4]), ptr(slots) if tokens else 0,
                   ptr(positions) if tokens else 0, ptr(result), stream)
    return [host(t) for t in (d[0], lens, cu, slots, positions, result)]


def table_case(rng, nseq, page, longest, most, pad=0, spare=0):
    cached = rng.integers(0, longest + 1, nseq)
    added = rng.integers(0, most + 1, nseq)
    have = -(-cached // page)
    R = int((-(-(cached + added) // page)).max()) + 1
    npages = int((-(-(cached + added) // page)).sum()) + 5
    order = rng.permutation(npages).astype(np.int32)
    bt = np.full((nseq, R), -1, np.int32)
    at = 0
    for s in range(nseq):
        bt[s, :have[s]] = order[at:at + have[s]]
        at += have[s]
    return bt, page, npages, int(added.sum()) + pad, cached, added, order, np.array([at, npages - spare])


@pytest.mark.parametrize("nseq, page, longest, most, pad", [
    (1, 16, 0, 1, 0), (1, 1, 0, 5000, 3), (3, 16, 40, 0, 2), (64, 16, 6000, 1, 0), (255, 24, 300, 90, 17), (256, 7, 100, 3, 0),
    (257, 16, 100, 200, 0), (1000, 128, 999, 40, 1000), (1025, 16, 64, 1, 0), (5000, 16, 50, 5, 7)])
def test_tables(nseq, page, longest, most, pad):
    rng = np.random.default_rng(nseq * 1000 + page)
    case = table_case(rng, nseq, page, longest, most, pad)
    for got, want, name in zip(run_tables(*case), pages_ref.tables(*case), ("bt", "lens", "cu", "slots", "positions", "result")):
        assert np.array_equal(got, want), name


@pytest.mark.parametrize("nseq", [5, 300])
def test_tables_of_steps_that_do_not_fit(nseq):
    """Too few free pages; lengths below zero and past a table; more tokens than places; pages outside the pool."""
    rng = np.random.default_rng(nseq)
    base = table_case(rng, nseq, 16, 100, 40)
    bt, page, npages, tokens, cached, added, free, span = base
    short = (bt, page, npages, tokens, cached, added, free, [span[0], span[0] + (span[1] - span[0]) // 3])
    none = (bt, page, npages, tokens, cached, added, free, [span[1], span[0]])
    c2, a2 = cached.copy(), added.copy()
    c2[0], a2[1], c2[2], c2[3] = -1, -7, bt.shape[1] * page, 2 ** 31 - 1
    a2[2], a2[3] = 1, 2 ** 31 - 1
    bad = (bt, page, npages, tokens, c2, a2, free, span)
    few = (bt, page, npages, tokens // 2, cached, added, free, span)
    nowhere = (bt, page, npages, 0, cached, added, free, span)
    b2 = bt.copy()
    b2[::2][b2[::2] >= 0] = npages + 3
    away = (b2, page, npages, tokens, cached, added, free, span)
    statuses = []
    for case in (short, none, bad, few, nowhere, away):
        want = pages_ref.tables(*case)
        statuses.append(int(want[5][1]))
        for got, w, name in zip(run_tables(*case), want, ("bt", "lens", "cu", "slots", "positions", "result")):
            assert np.array_equal(got, w), (name, statuses)
    assert statuses[0] & 1 and statuses[1] & 1 and statuses[2] & 2 and statuses[3] & 4 and statuses[4] & 4


# ---- append ----------------------------------------------------------------------------


def pool(rng, H, npages, page, D):
    """Codes and scales of one side; a NaN code here and there, as memory that nothing was written to has them."""
    codes = rng.integers(0, 256, (H, npages, page, D)).astype(np.uint8)
    scales = (0.002 + 0.02 * rng.random((H, npages))).astype(np.float16)
    return codes, scales


def run_append(sides, x, slots, page, stride=0, offset=0):
    """sides: ((codes, scales), (codes, scales)); x: (k, v) [tokens][H][D] float16."""
    c = w4amd.capi()
    H, npages, _, D = sides[0][0].shape
    d = [to_dev(a) for side in sides for a in side]
    row = stride or H * D
    flat = []
    for a in x:
        buf = np.zeros(len(a) * row + offset + 8, np.float16)
        for t in range(len(a)):
            buf[offset + t * row:offset + t * row + H * D] = a[t].ravel()
        flat.append(to_dev(buf))
    view = c.f8_pages_view(H, D, page, npages, *[ptr(t) for t in d])
    status = i32([0])
    c.quantize_f8_pages(view, ptr(flat[0]) + 2 * offset, ptr(flat[1]) + 2 * offset, stride, ptr(i32(slots)), len(slots), ptr(status))
    got = [host(t) for t in d]
    return [(got[0], got[1].view(np.float16)), (got[2], got[3].view(np.float16))], int(host(status)[0])


def slots_of(rng, lens, adds, page, pad=0):
    """Slots of sequences with lens[s] tokens in all, adds[s] of them new, on pages in arbitrary order."""
    need = [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + 2)
    slots, at = [], 0
    for n, a, k in zip(lens, adds, need):
        slots += [int(order[at + p // page]) * page + p % page for p in range(n - a, n)]
        at += k
    return np.array(slots + [-1] * pad, np.int32), len(order)


@pytest.mark.parametrize("H, D, page, lens, adds, stride, offset", [
    (1, 4, 1, [1], [1], 0, 0),
    (2, 64, 16, [5, 17, 33, 16], [1, 1, 1, 1], 0, 0),
    (3, 128, 16, [40, 100, 7], [40, 60, 1], 0, 0),
    (2, 128, 128, [300, 129], [290, 129], 1000, 0),
    (2, 256, 24, [100, 24, 25], [77, 24, 2], 0, 0),
    (1, 96, 7, [30, 1, 8], [29, 1, 3], 101, 0),
    (2, 20, 5, [23, 11], [9, 11], 0, 0),
    (2, 72, 16, [50, 20], [30, 4], 0, 1),
    (1, 512, 64, [200], [200], 0, 0),
    (2, 128, 1, [70, 3], [70, 2], 0, 0),
    (4, 64, 100, [1000], [950], 0, 0)])
def test_append(H, D, page, lens, adds, stride, offset):
    rng = np.random.default_rng(H * 10000 + D * 10 + page)
    slots, npages = slots_of(rng, lens, adds, page, pad=3)
    T = len(slots)
    # magnitudes over seven binades from token to token: scales of older pages have to rise
    x = [(rng.standard_normal((T, H, D)) * 2.0 ** rng.integers(-4, 4, (T, 1, 1))).astype(np.float16) for _ in range(2)]
    sides = [pool(rng, H, npages, page, D) for _ in range(2)]
    got, status = run_append(sides, x, slots, page, stride, offset)
    assert status == 0
    for (codes, scales), side, a in zip(got, sides, x):
        want_codes, want_scales, _ = pages_ref.append_side(*side, a, slots)
        assert np.array_equal(scales.view(np.uint16), want_scales.view(np.uint16))
        same(codes, want_codes)


def test_append_of_special_values():
    """All-zero pages, tokens that lift them, subnormal halves, infinities and NaN; padding and slots past the pool."""
    H, D, page, npages = 2, 64, 4, 9
    rng = np.random.default_rng(5)
    slots = np.array([0, 1, 5, 8, 9, -1, 12, 16, 17, 21, npages * page, 2 ** 31 - 1, -(2 ** 31), 24, 33], np.int32)
    x = [rng.standard_normal((len(slots), H, D)).astype(np.float16) for _ in range(2)]
    sides = [pool(rng, H, npages, page, D) for _ in range(2)]
    for a, (codes, scales) in zip(x, sides):
        a[0:2] = 0.0
        a[1, 0, 3] = -0.0
        scales[:, 1], codes[:, 1] = 0.0, 0       # an older page of zeros gets its first values
        a[3:5] = (rng.integers(-300, 300, (2, H, D)) * 2.0 ** -24).astype(np.float16)
        a[6, 0, :3] = [np.inf, -np.inf, np.nan]
        a[7, 1, 5] = np.inf
        a[8] = np.nan
        scales[:, 5] = np.float16(2.0 ** -24)    # older, tiny: lifted by many powers of two
        a[13] = np.float16(65504.0)
        scales[:, 8] = np.float16(1e-3)
        a[14] = 0.0                              # nothing to lift
    got, status = run_append(sides, x, slots, page)
    assert status == 1
    for (codes, scales), side, a in zip(got, sides, x):
        want_codes, want_scales, odd = pages_ref.append_side(*side, a, slots)
        assert odd and np.array_equal(scales.view(np.uint16), want_scales.view(np.uint16))
        same(codes, want_codes)


def test_append_every_half():
    """Every finite half as a quotient of several scales: the codes are the exactly rounded ones."""
    x = np.arange(1 << 16, dtype=np.uint16).view(np.float16)
    x = x[np.isfinite(x)]
    x = np.concatenate([x, np.zeros(-len(x) % 512, np.float16)]).reshape(-1, 1, 512)
    T = len(x)
    slots = 2 * np.arange(T, dtype=np.int32) + 1  # one older page of two rows each
    for top in (0.146, 3.3e-3, 147.0, 17.13):
        side = np.zeros((1, T, 2, 512), np.uint8), np.full((1, T), top, np.float16)
        got, _ = run_append([side, side], [x, x[::-1].copy()], slots, 2)
        for (codes, scales), a in zip(got, (x, x[::-1])):
            want_codes, want_scales, _ = pages_ref.append_side(*side, a, slots)
            same(scales, want_scales), same(codes, want_codes)


def test_append_in_steps_is_the_append_of_all():
    """Tokens one by one: no older value moves by more than the raised scale's subnormal step, and scales end at most a
    factor of two above those of one call."""
    rng = np.random.default_rng(11)
    H, D, page = 2, 64, 16
    x = [(rng.standard_normal((page, H, D)) * np.linspace(0.1, 3, page)[:, None, None]).astype(np.float16) for _ in range(2)]
    side = np.zeros((H, 1, page, D), np.uint8), np.zeros((H, 1), np.float16)
    once, _ = run_append([side, side], x, np.arange(page, dtype=np.int32), page)
    sides = [side, side]
    for t in range(page):
        sides, _ = run_append(sides, [a[t:t + 1] for a in x], np.array([t], np.int32), page)
    for (c1, s1), (c0, s0), a in zip(sides, once, x):
        s1, s0 = s1.astype(np.float64), s0.astype(np.float64)
        assert (s1 >= s0).all() and (s1 < 2 * s0 * (1 + 2 ** -10)).all()
        value = pages_ref.VALUES[c1[:, 0]] * s1[:, :, None]
        exact = a.astype(np.float64).transpose(1, 0, 2)
        # half a step of E4M3, and of its subnormals (2^-10) once for each time the scale was raised (at most 6: 30 x)
        assert (np.abs(value - exact) <= 2.0 ** -4 * np.abs(exact) + 6 * 2.0 ** -10 * s1[:, :, None]).all()


# ---- attention --------------------------------------------------------------------------


class Attn:
    """A cache of random codes with sequences on pages in arbitrary order; what lies past a sequence is NaN codes."""

    def __init__(self, seed, lens, adds, H, group, D, page, causal=True, holes=0, stride=0, scales=(0.002, 0.01), pad=0,
                 use_cu=True, max_len=None, max_q=None, q_scale=1.0, scale_spread=0):
        c = w4amd.capi()
        rng = np.random.default_rng(seed)
        self.args = H, group, D, page, causal
        self.lens, self.adds = np.array(lens), np.array(adds)
        need = [max(0, -(-n // page)) for n in lens]
        npages = sum(need) + 3
        order = rng.permutation(npages).astype(np.int32)
        R = max(need + [1]) + 1
        self.bt = rng.integers(0, npages, (len(lens), R)).astype(np.int32)
        written = np.zeros(npages * page, bool)
        at = 0
        for s, k in enumerate(need):
            self.bt[s, :k] = order[at:at + k]
            at += k
            t = np.arange(lens[s])
            written[self.bt[s, t // page] * page + t % page] = True
        self.k, self.v = [], []
        for side in (self.k, self.v):
            codes = pages_ref.encode(rng.standard_normal((H, npages * page, D)) * 100)
            codes[:, ~written] = 0x7F
            z = scales[0] + scales[1] * rng.random((H, npages))
            if scale_spread:
                z = z * 2.0 ** rng.integers(-scale_spread, scale_spread + 1, (H, npages))
            side += [codes.reshape(H, npages, page, D), z.astype(np.float16)]
        if holes:  # pages that were given back
            for s, k in enumerate(need):
                for j in rng.integers(0, max(k, 1), holes):
                    self.bt[s, j] = rng.choice([-1, npages, 2 ** 31 - 1, -(2 ** 31)])
        T = int(sum(adds)) + pad
        self.q = (rng.standard_normal((T, H * group, D)) * q_scale).astype(np.float16)
        self.cu = np.concatenate([[0], np.cumsum(adds)]).astype(np.int32) if use_cu else None
        row = H * group * D
        self.row = stride or row
        q = np.full(T * self.row, np.nan, np.float16)
        for t in range(T):
            q[t * self.row:t * self.row + row] = self.q[t].ravel()
        self.d = [to_dev(a) for a in (q, self.k[0], self.k[1], self.v[0], self.v[1])] + [i32(self.bt), i32(self.lens)]
        self.cu_d = i32(self.cu) if use_cu else None
        self.view = c.f8_pages_view(H, D, page, npages, *[ptr(t) for t in self.d[1:5]])
        self.batch = c.paged_batch(len(lens), T, max_q or max(1, int(max(adds))), max_len or max(1, int(max(lens))),
                                   ptr(self.d[5]), R, ptr(self.d[6]), ptr(self.cu_d))
        self.before = np.full((T, H * group, D), 7.0, np.float16)
        n = c.attention_f8_pages_workspace(self.view, self.batch, group)
        self.space = torch.zeros(n + 16, dtype=torch.uint8, device=DEV)
        self.n, self.stride, self.npages = n, stride, npages

    def run(self, stream=0, out=None, space=None):
        H, group, D, page, causal = self.args
        out = to_dev(self.before) if out is None else out
        w4amd.capi().attention_f8_pages(self.view, self.batch, group, causal, ptr(self.d[0]), self.stride, ptr(out),
                                        ptr(self.space if space is None else space), self.n, stream)
        return out

    def want(self):
        H, group, D, page, causal = self.args
        return pages_ref.attention(self.q, self.bt, self.lens, self.cu, self.k, self.v, page, self.npages, group, causal, self.before)

    def check(self, out=None):
        got = host(self.run() if out is None else out).view(np.float16).reshape(self.before.shape).astype(np.float64)
        want, tol = self.want()
        off = np.abs(got - want)
        assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), np.argwhere(~(off <= tol))[:4].tolist())
        return got


@pytest.mark.parametrize("D", [64, 96, 128, 256, 4, 20, 80, 512])
@pytest.mark.parametrize("page", [1, 7, 16, 24, 128])
def test_decode(D, page):
    Attn(D + page, [1, 15, 16, 17, 129, 300], [1] * 6, 2, 3, D, page).check()


@pytest.mark.parametrize("group", [1, 2, 4, 7, 8, 16, 17, 32, 64])
def test_decode_groups(group):
    Attn(group, [1, 40, 200], [1, 1, 1], 2, group, 64, 16).check()


@pytest.mark.parametrize("H, group, D, page, L", [(1, 4, 128, 16, 4097), (2, 1, 64, 16, 9000), (1, 8, 256, 64, 3000),
                                                  (1, 2, 96, 24, 5001), (1, 3, 128, 1, 2500), (1, 2, 40, 16, 3100)])
def test_decode_in_splits(H, group, D, page, L):
    """Long caches are cut over workgroups; short ones beside them are not."""
    Attn(L, [L, 3, L // 2 + 1, 0, 700], [1, 1, 1, 0, 1], H, group, D, page).check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 7, 24), (256, 1, 64), (96, 16, 16), (36, 2, 5)])
def test_a_few_tokens(causal, D, group, page):
    Attn(D * group, [5, 300, 77, 33, 1], [5, 3, 1, 0, 1], 2, group, D, page, causal).check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 7, 24), (256, 2, 64), (96, 3, 16), (128, 1, 1)])
def test_prompts(causal, D, group, page):
    Attn(D * group + 1, [131, 400, 64, 90], [131, 150, 63, 0], 1, group, D, page, causal).check()


def test_prompts_next_to_decoding_sequences():
    Attn(3, [700, 1200, 30, 5, 900], [300, 1, 1, 5, 1], 2, 4, 128, 16, pad=9).check()


def test_long_context_prompt_in_splits():
    Attn(4, [5000], [40], 1, 4, 128, 16).check()


@pytest.mark.parametrize("adds", [[1, 1, 1], [4, 3, 1], [90, 40, 200]])
def test_pages_that_were_given_back(adds):
    """Table entries outside the pool are positions that nobody sees."""
    a = Attn(sum(adds), [300, 90, 260], adds, 2, 4, 128, 16, holes=6)
    a.check()
    a.bt[1] = -1  # a sequence that has none left
    a.d[5].copy_(i32(a.bt))
    got = a.check()
    assert (got[a.cu[1]:a.cu[2]] == 0).all()


@pytest.mark.parametrize("lens, adds", [([0, 5], [1, 1]), ([3, 40], [8, 8]), ([0, 0], [70, 2]), ([30, 200], [100, 150])])
def test_queries_that_see_nothing(lens, adds):
    """More queries than positions: the first of them lie before position 0."""
    got = Attn(sum(lens) + 1, lens, adds, 2, 4, 64, 16).check()
    assert (got[:max(0, adds[0] - lens[0])] == 0).all()


@pytest.mark.parametrize("adds", [[1, 1], [3, 2], [80, 1]])
def test_one_token_per_sequence_strides_padding_and_bounds(adds):
    a = Attn(8, [100, 260], adds, 2, 2, 128, 16, stride=1000, pad=5)
    got = a.check()
    assert (got[sum(adds):] == 7.0).all()
    if adds == [1, 1]:
        Attn(9, [100, 260, 0], [1, 1, 1], 2, 2, 128, 16, use_cu=False).check()
        Attn(9, [100, 260], adds, 2, 2, 128, 16, max_len=5000).check()  # longer than any of them is
    Attn(10, [100, 260], adds, 2, 2, 128, 16, stride=1001).check()       # rows at odd addresses


def test_lengths_past_the_bounds_of_a_call_are_cut():
    """max_len and the tables bound what is read, whatever lens says."""
    a = Attn(12, [100, 260], [1, 1], 2, 2, 128, 16, max_len=128)
    a.lens = np.array([100, 260])
    out = a.run()
    a.lens = np.array([100, 128])
    a.args = (*a.args[:4], False)  # (the second sequence's query still lies past what is kept)
    a.check(out)
    b = Attn(13, [100, 260], [1, 1], 2, 2, 128, 16)
    b.d[6].copy_(i32([2 ** 31 - 1, -(2 ** 31)]))
    host(b.run())


@pytest.mark.parametrize("adds", [[1, 1, 1], [3, 1, 2], [120, 1, 64]])
def test_scales_far_apart(adds):
    """Page scales over 2^20 to both sides, values that would leave FP16 as weights."""
    Attn(21, [300, 50, 128], adds, 1, 4, 128, 16, scale_spread=9).check()
    Attn(22, [300, 50, 128], adds, 1, 4, 64, 16, scales=(2.0 ** -22, 2.0 ** -22)).check()
    a = Attn(23, [300, 50, 128], adds, 1, 4, 128, 16)
    for side in (a.k, a.v):
        side[1][:, ::2] = 0.0  # pages of zeros
    a.d[2].copy_(to_dev(a.k[1])), a.d[4].copy_(to_dev(a.v[1]))
    a.check()


def test_peaked_and_flat_scores():
    Attn(31, [700, 3], [1, 1], 1, 4, 128, 16, q_scale=30.0).check()
    Attn(32, [700, 90], [1, 70], 1, 4, 128, 16, q_scale=30.0).check()
    Attn(33, [700, 90], [1, 70], 1, 4, 128, 16, q_scale=0.0).check()


@pytest.mark.parametrize("adds", [[1, 1], [40, 40]])
def test_nan_of_one_query_stays_its_own(adds):
    a = Attn(41, [200, 90], adds, 2, 4, 128, 16)
    clean = host(a.run()).copy()
    q = a.q.copy()
    q[0, 1, 5] = np.nan
    a.d[0].copy_(to_dev(q).view(-1))
    got = host(a.run()).view(np.float16).reshape(a.before.shape)
    assert np.isnan(got[0, 1]).all()
    keep = np.ones(got.shape[:2], bool)
    keep[0, 1] = False
    assert np.array_equal(got[keep].view(np.uint16), clean.view(np.uint16).reshape(got.shape)[keep])


@pytest.mark.parametrize("nseq", [64, 65, 200, 256, 257])
@pytest.mark.parametrize("longest", [300, 2600])
def test_many_sequences(nseq, longest):
    """One long sequence among many short ones, some without tokens or positions."""
    rng = np.random.default_rng(nseq)
    lens, adds = rng.integers(0, 40, nseq), np.ones(nseq, np.int64)
    lens[nseq // 2], lens[3], adds[5] = longest, 0, 0
    Attn(nseq + longest, lens.tolist(), adds.tolist(), 1, 2, 64, 16).check()
    if longest > 300:
        adds[7:9], lens[7:9] = 5, 900
        Attn(nseq, lens.tolist(), adds.tolist(), 1, 4, 64, 16).check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group, adds", [(33, [1, 1, 1]), (64, [1, 0, 1]), (4, [9, 16, 8]), (1, [33, 32, 65]), (7, [40, 1, 11])])
def test_blocks_of_rows_in_splits(D, group, adds):
    """More rows of a KV head than a workgroup takes, on caches that are cut over workgroups."""
    Attn(D + group, [1900, 20, 700], adds, 1, group, D, 16).check()


@pytest.mark.parametrize("adds", [[30, 21], [700, 90]])
@pytest.mark.parametrize("page", [1, 3, 16])
def test_a_call_of_either_kernel(adds, page):
    """The same rows by one kernel, and by the other where the bounds of the call are far off."""
    lens = [max(900, adds[0]), 200]
    a = Attn(71, lens, adds, 1, 8, 128, page)
    b = Attn(71, lens, adds, 1, 8, 128, page, max_q=adds[0] + 1000, max_len=10 ** 6)
    a.check(), b.check()


@pytest.mark.parametrize("nseq", [3, 70, 260])
@pytest.mark.parametrize("D, group, page", [(64, 7, 16), (96, 4, 32), (128, 4, 16), (256, 2, 16), (128, 20, 16), (64, 4, 24)])
def test_chunks_next_to_decoding_sequences(D, group, page, nseq):
    """Calls whose bounds are past what one kernel takes alone; prompts, single tokens and idle sequences side by side."""
    rng = np.random.default_rng(D + nseq)
    lens, adds = rng.integers(1, 200, nseq), np.ones(nseq, np.int64)
    lens[:3], adds[:3] = [1400, 900, 260], [130, 1, 70]
    if nseq > 3:
        adds[5], lens[9], adds[9] = 0, 1700, 16 // group + 1
    Attn(nseq + D, lens.tolist(), adds.tolist(), 1, group, D, page, pad=6000).check()


def test_batches_of_every_kind_in_one_workspace():
    """Whatever a call leaves in the workspace, the next one of another shape finds what it needs."""
    kinds = [([3000, 40], [1, 1], 2, 4, 128, 16), ([900, 800], [200, 1], 1, 4, 128, 16), ([5000], [2], 1, 7, 64, 24),
             ([400] * 70, [1] * 70, 1, 1, 96, 16), ([2100], [1], 1, 1, 40, 16), ([700, 2000], [40, 33], 1, 2, 256, 64)]
    calls = [Attn(80 + i, *k) for i, k in enumerate(kinds)]
    want = [host(x.run()).copy() for x in calls]
    space = torch.zeros(max(x.n for x in calls) + 16, dtype=torch.uint8, device=DEV)
    order = np.random.default_rng(1).integers(0, len(calls), 60)
    outs = [calls[i].run(space=space) for i in order]
    assert all(np.array_equal(host(o), want[i]) for o, i in zip(outs, order))
    for x in calls:
        x.check()


def test_more_rows_than_workgroups():
    """Every row's only position is the first: its V."""
    a = Attn(90, [1], [1], 2, 1, 4, 1, causal=False)
    c, T, group = w4amd.capi(), 16500, 32
    q = torch.zeros(T * 2 * group * 4, dtype=torch.float16, device=DEV)
    out = torch.zeros_like(q)
    cu = i32([0, T])
    batch = c.paged_batch(1, T, T, 1, ptr(a.d[5]), a.bt.shape[1], ptr(a.d[6]), ptr(cu))
    assert c.attention_f8_pages_workspace(a.view, batch, group) == 0
    c.attention_f8_pages(a.view, batch, group, 0, ptr(q), 0, ptr(out))
    got = out.cpu().numpy().reshape(T, 2, group, 4)
    exact = pages_ref.VALUES[a.v[0][:, a.bt[0, 0], 0]] * a.v[1][:, a.bt[0, 0]].astype(np.float64)[:, None]
    assert (np.abs(got - exact[None, :, None]) <= 2.0 ** -10 * np.abs(exact)[None, :, None]).all()


@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 7, 24), (256, 2, 64), (96, 16, 16), (128, 8, 1), (40, 2, 5)])
@pytest.mark.parametrize("lens, adds", [([40, 33, 5], [4, 1, 5]), ([50, 300], [45, 150]), ([3000, 70], [1500, 70])])
def test_nan_codes_reach_only_the_rows_that_see_them(D, group, page, lens, adds):
    """A cached NaN makes NaN of its column (of V) or row (of K) where a causal query sees it, and of nothing else."""
    if D == 40 and lens[0] == 3000:
        lens, adds = [600, 70], [300, 70]
    a = Attn(D + group, lens, adds, 1, group, D, page)
    rng = np.random.default_rng(7)
    for s, (n, m) in enumerate(zip(lens, adds)):
        for back in {1, 2, max(1, m // 2), max(1, m - 1)}:  # among the last m tokens
            t = n - back
            row = a.bt[s, t // page] * page + t % page
            a.v[0].reshape(-1, D)[row, rng.integers(0, D, 2)] = [0x7F, 0xFF]
        if s == 1:
            row = a.bt[s, (n - 2) // page] * page + (n - 2) % page
            a.k[0].reshape(-1, D)[row, 3] = 0x7F
    a.d[1].copy_(to_dev(a.k[0]).view(a.d[1].shape)), a.d[3].copy_(to_dev(a.v[0]).view(a.d[3].shape))
    got = host(a.run()).view(np.float16).reshape(a.before.shape).astype(np.float64)
    want, tol = a.want()
    nan = np.isnan(want)
    assert nan.any() and not nan.all()
    assert np.array_equal(np.isnan(got), nan), np.argwhere(np.isnan(got) != nan)[:4].tolist()
    off = np.abs(got - want)[~nan]
    assert (off <= tol[~nan]).all()


# ---- use ---------------------------------------------------------------------------------


@pytest.mark.parametrize("adds", [[1, 1, 1, 1], [300, 1, 4, 40]])
def test_calls_repeat_their_bytes_and_leave_the_workspace_ready(adds):
    a = Attn(51, [3000, 800, 5000, 40], adds, 1, 4, 128, 16)
    first = host(a.run()).copy()
    for _ in range(3):
        assert np.array_equal(host(a.run()), first)


def test_two_streams_with_workspaces_of_their_own():
    a, b = Attn(61, [5000, 100], [1, 1], 1, 4, 128, 16), Attn(62, [3000, 4000], [1, 30], 1, 4, 128, 16)
    want = [host(x.run()).copy() for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(5):
        for x, s, o in zip((a, b), streams, outs):
            with torch.cuda.stream(s):
                o.append(to_dev(x.before))
                x.run(s.cuda_stream, o[-1])
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(np.array_equal(host(t), w) for t in o)


class Step:
    """A serving loop's state: tables, cache and buffers that every step uses."""

    def __init__(self, seed, nseq, H, group, D, page, npages, R, tokens, max_q):
        c = w4amd.capi()
        self.rng = np.random.default_rng(seed)
        self.H, self.group, self.D, self.page, self.npages, self.tokens = H, group, D, page, npages, tokens
        self.bt = np.full((nseq, R), -1, np.int32)
        self.lens = np.zeros(nseq, np.int64)
        self.free = self.rng.permutation(npages).astype(np.int32)
        self.taken = 0
        self.k = self.v = (np.full((H, npages, page, D), 0x7F, np.uint8), np.zeros((H, npages), np.float16))
        self.d = {n: i32(a) for n, a in (("bt", self.bt), ("cached", self.lens), ("added", self.lens), ("free", self.free),
                                         ("span", [0, npages]), ("lens", self.lens), ("cu", np.zeros(nseq + 1)),
                                         ("slots", np.zeros(tokens)), ("positions", np.zeros(tokens)), ("result", [0, 0]),
                                         ("status", [0]))}
        self.pool = [to_dev(a) for a in (*self.k, *self.v)]
        self.row = (group + 2) * H * D
        self.qkv = to_dev(np.zeros((tokens, self.row), np.float16))
        self.out = to_dev(np.zeros((tokens, H * group, D), np.float16))
        self.view = c.f8_pages_view(H, D, page, npages, *[ptr(t) for t in self.pool])
        self.batch = c.paged_batch(nseq, tokens, max_q, R * page, ptr(self.d["bt"]), R, ptr(self.d["lens"]), ptr(self.d["cu"]))
        self.n = c.attention_f8_pages_workspace(self.view, self.batch, group)
        self.space = torch.zeros(self.n + 16, dtype=torch.uint8, device=DEV)

    def launch(self, stream=0):
        c, d = w4amd.capi(), {n: ptr(t) for n, t in self.d.items()}
        at = self.qkv.data_ptr()
        c.paged_tables(self.batch, self.page, self.npages, d["cached"], d["added"], d["free"], d["span"], d["slots"],
                       d["positions"], d["result"], stream)
        k = at + 2 * self.group * self.H * self.D
        c.quantize_f8_pages(self.view, k, k + 2 * self.H * self.D, self.row, d["slots"], self.tokens, d["status"], stream)
        c.attention_f8_pages(self.view, self.batch, self.group, 1, at, self.row, ptr(self.out), ptr(self.space), self.n, stream)

    def step(self, added, go):
        """One step with new inputs; `go` launches it.  Everything is compared with the definitions."""
        H, g, D = self.H, self.group, self.D
        qkv = (self.rng.standard_normal((self.tokens, self.row)) * 2.0 ** self.rng.integers(-2, 3, (self.tokens, 1))).astype(np.float16)
        self.qkv.copy_(to_dev(qkv))
        self.d["cached"].copy_(i32(self.lens))
        self.d["added"].copy_(i32(added))
        self.d["span"].copy_(i32([self.taken, self.npages]))
        self.out.fill_(0)
        go()
        bt, lens, cu, slots, positions, result = pages_ref.tables(self.bt, self.page, self.npages, self.tokens, self.lens, added,
                                                                  self.free, [self.taken, self.npages])
        for name, want in (("bt", bt), ("lens", lens), ("cu", cu), ("slots", slots), ("positions", positions), ("result", result)):
            assert np.array_equal(host(self.d[name]), want), name
        rows = qkv.reshape(self.tokens, g + 2, H, D)
        self.k, self.v = (pages_ref.append_side(*side, rows[:, g + i], slots)[:2] for i, side in enumerate((self.k, self.v)))
        for got, want in zip(self.pool, (*self.k, *self.v)):
            got = host(got)
            assert np.array_equal(got.view(want.dtype) if want.dtype == np.float16 else got, want)
        q = qkv[:, :g * H * D].reshape(self.tokens, g * H, D)
        want, tol = pages_ref.attention(q, bt, lens, cu, self.k, self.v, self.page, self.npages, g, True,
                                        np.zeros((self.tokens, g * H, D)))
        off = np.abs(host(self.out).view(np.float16).reshape(want.shape).astype(np.float64) - want)
        assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())
        self.bt, self.lens, self.taken = bt, lens.astype(np.int64), self.taken + int(result[0])
        return result


def test_prompts_then_decode():
    """Prompts of three sequences, then tokens one by one, one sequence idle for a while, then a chunk."""
    s = Step(71, 3, 2, 4, 64, 16, 40, 12, 120, 100)
    for added in ([50, 17, 1], [1, 1, 1], [1, 0, 1], [1, 1, 1], [4, 90, 1], [1, 1, 1]):
        assert s.step(np.array(added), s.launch)[1] == 0
    assert s.step(np.array([100, 0, 5]), s.launch)[1] == 0  # (58 + 100 tokens: a table holds 12 pages of 16)
    assert s.step(np.array([100, 1, 5]), s.launch)[1] == 2  # past the first one's table: the others go on
    assert s.step(np.array([1, 1, 1]), s.launch)[1] == 0


def test_a_captured_step_replayed():
    """The whole step as a graph: lengths, pages and sizes change between the replays, the launches do not."""
    s = Step(72, 4, 1, 4, 128, 16, 60, 40, 70, 64)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.launch(side.cuda_stream)

    def replay():
        graph.replay()
        torch.cuda.synchronize()

    for added in ([64, 3, 1, 0], [1, 1, 1, 1], [2, 40, 0, 20], [1, 1, 1, 1]):
        s.step(np.array(added), replay)
        torch.ones(1000, device=DEV).sum().item()  # the program's own work between replays
    s.step(np.array([1, 1, 1, 1]), s.launch)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes a side, sequences on its last pages."""
    c = w4amd.capi()
    H, D, page, npages = 2, 128, 64, 300_000
    rng = np.random.default_rng(81)
    q_k = torch.zeros(H, npages, page, D, dtype=torch.uint8, device=DEV)
    q_v = torch.zeros_like(q_k)
    s_k = torch.zeros(H, npages, dtype=torch.float16, device=DEV)
    s_v = torch.zeros_like(s_k)
    assert q_k[0].numel() > 1 << 31 and q_k.numel() > 1 << 32
    ids = np.array([[npages - 1, 3], [npages - 2, npages - 3]], np.int32)
    lens, adds = np.array([100, 128]), np.array([100, 128])
    view = c.f8_pages_view(H, D, page, npages, ptr(q_k), ptr(s_k), ptr(q_v), ptr(s_v))
    T = 228
    x = [rng.standard_normal((T, H, D)).astype(np.float16) for _ in range(2)]
    slots = np.concatenate([ids[s, np.arange(n) // page] * page + np.arange(n) % page for s, n in enumerate(lens)]).astype(np.int32)
    xd, status = [to_dev(a) for a in x], i32([0])
    c.quantize_f8_pages(view, ptr(xd[0]), ptr(xd[1]), 0, ptr(i32(slots)), T, ptr(status))
    small = {int(p): i for i, p in enumerate(ids.ravel())}  # the pages in use, as a pool of their own
    sides = []
    for codes, scales, a in ((q_k, s_k, x[0]), (q_v, s_v, x[1])):
        want = pages_ref.append_side(np.zeros((H, 4, page, D), np.uint8), np.zeros((H, 4), np.float16), a,
                                     np.array([small[int(t) // page] * page + int(t) % page for t in slots], np.int32))[:2]
        at = torch.from_numpy(ids.ravel().astype(np.int64)).to(DEV)
        assert np.array_equal(host(codes[:, at]), want[0]) and np.array_equal(host(scales[:, at]), want[1])
        sides.append(want)
    for n in ([100, 128], [1, 1], [5, 9]):
        cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        q = rng.standard_normal((int(cu[-1]), H * 2, D)).astype(np.float16)
        out = to_dev(np.zeros(q.shape, np.float16))
        bt_d, lens_d, cu_d, q_d = i32(ids), i32(lens), i32(cu), to_dev(q)
        batch = c.paged_batch(2, len(q), max(n), 128, ptr(bt_d), 2, ptr(lens_d), ptr(cu_d))
        size = c.attention_f8_pages_workspace(view, batch, 2)
        space = torch.zeros(size + 16, dtype=torch.uint8, device=DEV)
        c.attention_f8_pages(view, batch, 2, 1, ptr(q_d), 0, ptr(out), ptr(space), size)
        want, tol = pages_ref.attention(q, np.vectorize(small.get)(ids), lens, cu, *sides, page, 4, 2, True, np.zeros(q.shape))
        got = host(out).view(np.float16).reshape(q.shape).astype(np.float64)
        assert (np.abs(got - want) <= tol).all()


def test_serving_through_the_cpp_api():
    from test_cpp_gates import _run
    assert " 0 failures" in _run("test_pages", 100)
