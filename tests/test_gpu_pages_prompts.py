"""Paged FP8 attention where tests of small calls do not reach: the kernel for many rows, by calls whose bounds are past what
the one for few rows takes, far positions, values that are not finite."""
import numpy as np
import pytest
import torch

import pages_ref
import w4amd
from devutil import DEV, ptr, to_dev
from test_gpu_pages import Attn, Step, host, i32

pytestmark = pytest.mark.gpu

FEW_WORK = 7e8  # rows of a call times positions times D, up to which the other kernel takes everything


def prompts(seed, lens, adds, H, group, D, page, **more):
    """Places behind the last sequence until the call is one of the kernel for many rows."""
    longest = min(more.get("max_len") or max(lens), (max(-(-max(lens) // page), 1) + 1) * page)
    pad = max(0, int(FEW_WORK / (H * group * longest * D)) + 1 - sum(adds))
    a = Attn(seed, lens, adds, H, group, D, page, pad=pad, **more)
    a.plan = w4amd.capi().attention_f8_pages_plan_for(a.view, a.batch, group)
    assert a.plan[0] >= 2 and any(n * group > a.plan[1] for n in adds), a.plan
    return a


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [1, 7, 24])
def test_pages_that_are_no_multiple_of_16(D, page):
    """Tiles whose scales are laid out by the four waves; with pages of one position a table holds 448 of them, and what
    is left over is a single tile."""
    prompts(D + page, [449, 512, 64, 40, 960], [120, 64, 64, 33, 50], 1, 4, D, page).check()
    prompts(D + page + 1, [64], [64], 2, 4, D, page).check()
    prompts(D + page + 2, [500], [90], 1, 4, D, page).check()


# ---- far positions -------------------------------------------------------------------------


def with_tables(a, bt, max_len, lens=None):
    """The calls of `a` with other tables, a bound and lengths."""
    c = w4amd.capi()
    H, group, D, page, causal = a.args
    a.bt, a.d[5] = bt, i32(bt)
    if lens is not None:
        a.lens, a.d[6] = np.array(lens), i32(lens)
    a.batch = c.paged_batch(len(bt), len(a.q), int(max(a.adds)), max_len, ptr(a.d[5]), bt.shape[1], ptr(a.d[6]), ptr(a.cu_d))
    a.n = c.attention_f8_pages_workspace(a.view, a.batch, group)
    a.space = torch.zeros(a.n + 16, dtype=torch.uint8, device=DEV)
    return a


@pytest.mark.parametrize("adds", [[1, 1], [5, 2], [300, 1], [90, 64]])
@pytest.mark.parametrize("D", [128, 40])
def test_short_sequences_under_the_largest_bound(D, adds):
    """Tables and a bound of 2^30 positions: prompts and single tokens are computed as under a bound of their own."""
    a = Attn(D, [400, 200], adds, 1, 4, D, 1024)
    bt = np.full((2, 1 << 20), -1, np.int32)
    bt[:, :a.bt.shape[1]] = a.bt
    with_tables(a, bt, 2 ** 31 - 1).check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_the_longest_sequence(causal, n):
    """2^30 - 3 positions whose table names page 0 in its first half, page 1 in its second and page 2 at its end.  Scores are
    0 but for the last page, whose 2^20 positions (three of them behind the end) have as much weight as all others."""
    H, group, D, page = 1, 4, 64, 1 << 20
    L = (1 << 30) - 3
    a = Attn(7, [64], [n], H, group, D, 64, causal)
    a.args, entries = (H, group, D, page, causal), 1 << 10
    q = np.zeros_like(a.q)
    q[..., 0] = 8.0
    codes = [np.zeros((H, 3, page, D), np.uint8) for _ in range(2)]
    codes[0][:, 2, :, 0] = 0x38                            # 1
    for p, one in enumerate((0x38, 0x40, 0x48)):           # 1, 2, 4
        codes[1][:, p] = one
    # 8 sk / sqrt(64) nats; (2^30 - 2^20) / 2^20 = 1023 times as many others
    sk = float(np.float16(np.log(1023)))
    scales = [np.full((H, 3), sk, np.float16), np.ones((H, 3), np.float16)]
    a.k, a.v = [codes[0], scales[0]], [codes[1], scales[1]]
    a.d[0:5] = [to_dev(x) for x in (q, codes[0], scales[0], codes[1], scales[1])]
    c = w4amd.capi()
    a.view = c.f8_pages_view(H, D, page, 3, *[ptr(t) for t in a.d[1:5]])
    bt = np.repeat(np.array([0, 1], np.int32), entries // 2)
    bt[-1] = 2
    with_tables(a, bt[None], L, [L])
    got = host(a.run()).view(np.float16).reshape(q.shape).astype(np.float64)
    half = entries // 2 * page
    for i in range(n):
        last = (L - n + i + 1 if causal else L) - (entries - 1) * page
        w = np.array([half, half - page, last * np.exp(sk)])
        want = w @ np.array([1.0, 2.0, 4.0]) / w.sum()
        # A lane adds its weights, and a matrix product its sums, at most 2^17 times (2^30 positions over 512 workgroups in
        # tiles of 64, four additions each); an addition is off by 2^-24 of the sum.  Weights and the output are halves.
        assert (np.abs(got[i] - want) <= want * (2 * 2.0 ** (17 - 24) + 2.0 ** -10)).all(), (i, got[i].min(), got[i].max(), want)


# ---- NaN codes -----------------------------------------------------------------------------


def with_nan_codes(a, rng):
    """NaN codes of V in every second page of each sequence and in one of its last tokens, half of these pages under a scale
    of 0; codes of K under a scale of 0."""
    H, group, D, page, _ = a.args
    for s, (n, m) in enumerate(zip(a.lens, a.adds)):
        for j, t in enumerate([*range(page // 2, n - m, 2 * page)][:3] + [n - m // 2 - 1]):
            pg = a.bt[s, t // page]
            a.v[0][rng.integers(H), pg, t % page, rng.integers(0, D, 2)] = [0x7F, 0xFF]
            if j % 2 == s % 2:
                a.v[1][:, pg] = 0.0
    a.k[1][:, a.bt[0, 0]] = 0.0
    for at, x in ((2, a.k[1]), (3, a.v[0]), (4, a.v[1])):
        a.d[at].copy_(to_dev(x).view(a.d[at].shape))
    return a


def check_nan(a):
    got = host(a.run()).view(np.float16).reshape(a.before.shape).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, tol = a.want()
    nan = np.isnan(want)
    assert nan.any() and not nan.all()
    assert np.array_equal(np.isnan(got), nan), np.argwhere(np.isnan(got) != nan)[:4].tolist()
    assert (np.abs(got - want)[~nan] <= tol[~nan]).all()


@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 7, 24), (256, 2, 64), (96, 16, 16), (128, 8, 1), (40, 2, 5)])
@pytest.mark.parametrize("lens, adds", [([40, 333, 5], [1, 1, 1]), ([50, 600], [5, 3]), ([300, 170], [60, 80])])
def test_nan_codes_under_a_scale_of_0(D, group, page, lens, adds):
    """A NaN stays one under a scale of 0, wherever in a tile it stands and whichever kernel reads it."""
    check_nan(with_nan_codes(Attn(D, lens, adds, 2, group, D, page), np.random.default_rng(3)))
    if D != 40 and max(adds) > 1:
        many = [n * 40 // max(adds) for n in adds] if max(adds) < 40 else adds
        check_nan(with_nan_codes(prompts(D, lens, many, 2, group, D, page), np.random.default_rng(4)))


# ---- kernels side by side ------------------------------------------------------------------


@pytest.mark.parametrize("nseq, H, kind", [(255, 8, 4), (256, 8, 4), (257, 8, 3), (256, 16, 3)])
def test_many_sequences_next_to_a_chunk(nseq, H, kind):
    """One launch with workgroups for half of the card, for all of it, and two launches."""
    rng = np.random.default_rng(nseq)
    lens, adds = rng.integers(1, 30, nseq), np.ones(nseq, np.int64)
    lens[3], adds[3], lens[100], adds[7] = 600, 40, 500, 0
    a = prompts(nseq, lens.tolist(), adds.tolist(), H, 1, 64, 16)
    assert a.plan[0] == kind
    a.check()
    first = host(a.run()).copy()
    assert np.array_equal(host(a.run()), first)


# ---- weights far apart ---------------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n, many", [(1, False), (5, False), (20, False), (60, True)])
def test_small_weights_next_to_a_token_without_values(D, n, many):
    """A first token that takes nearly all of the softmax and has no values (an attention sink): the others, 2^25 to 2^27
    times below it, are all of the output."""
    a = (prompts if many else Attn)(D + n, [400], [n], 1, 4, D, 16)
    H, group, D, page, _ = a.args
    rng = np.random.default_rng(n)
    first = a.bt[0, 0]
    a.q[...] = 0
    a.q[..., 0] = np.sqrt(D)
    a.q[..., 1] = np.sqrt(D) / 16
    a.k[0][...] = 0
    a.k[0][0, first, 0, 0] = 0x38                                                        # 1: sk nats
    a.k[0][..., 1] = rng.choice(np.array([0x00, 0x38, 0xB8], np.uint8), a.k[0].shape[:3])  # 0, 1, -1: sk / 16 nats = 1.6 binades
    a.k[1][...] = np.float16(26 * np.log(2))
    a.v[0][...] = pages_ref.encode(100 + 100 * rng.random(a.v[0].shape))
    a.v[0][0, first, 0] = 0
    a.v[1][...] = 1.0
    q = np.zeros((len(a.q), a.row), np.float16)
    q[:] = a.q.reshape(len(a.q), -1)
    for at, x in ((0, q), (1, a.k[0]), (2, a.k[1]), (3, a.v[0]), (4, a.v[1])):
        a.d[at].copy_(to_dev(x).view(a.d[at].shape))
    got = host(a.run()).view(np.float16).reshape(a.before.shape).astype(np.float64)[:n]
    want = a.want()[0][:n]
    # Weights are kept at 2^6 times what they are to the largest one, so those below halves' normal range are off by 2^-31 of
    # that at most; values are positive and at most 200.  Others' are rounded by 2^-11, as is the output; exponents of up to 26
    # are off by 2^-21 times 26.
    assert (want > 1e-4).all()
    assert (np.abs(got - want) <= 2.0 ** -31 * 400 * 200 + (2.0 ** -10 + 2.0 ** -16) * want).all(), float((np.abs(got - want) / want).max())


# ---- the kernel for many rows on what tests of small calls give the one for few -------------

SHAPES = [(128, 4, 16), (64, 7, 24), (256, 2, 64), (96, 3, 16), (128, 1, 1), (96, 5, 7), (256, 4, 24), (64, 1, 16), (128, 40, 16)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D, group, page", SHAPES)
def test_prompts_of_any_length(D, group, page, causal):
    prompts(D * group + page, [131, 400, 64, 90], [131, 150, 63, 0], 1, group, D, page, causal=causal).check()
    prompts(D * group + page + 1, [777], [1 + 40 // group], 2, group, D, page, causal=causal).check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D, group, page", SHAPES)
def test_prompts_over_pages_that_were_given_back(D, group, page, causal):
    """Table entries outside the pool, in the first tile and the last, all of a sequence's, and next to scales of 0."""
    a = prompts(D + group, [300, 290, 260], [90, 40, 200], 1, group, D, page, causal=causal, holes=2 + 40 // page)
    a.check()
    a.bt[1] = -1                                        # a sequence that has none left
    a.bt[0, 0] = a.bt[0, 299 // page] = a.npages
    a.d[5].copy_(i32(a.bt))
    got = a.check()
    assert (got[a.cu[1]:a.cu[2]] == 0).all()
    for side in (a.k, a.v):
        side[1][:, ::2] = 0.0
    a.d[2].copy_(to_dev(a.k[1])), a.d[4].copy_(to_dev(a.v[1]))
    a.check()


@pytest.mark.parametrize("lens, adds", [([3, 40], [50, 48]), ([0, 45], [70, 40]), ([0, 400], [70, 1]), ([30, 200], [100, 250])])
@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 2, 24), (256, 1, 16), (96, 8, 1)])
def test_prompts_that_see_nothing(D, group, page, lens, adds):
    """More queries than positions: the first of them lie before position 0; sequences without any."""
    got = prompts(sum(lens) + D, lens, adds, 2, group, D, page).check()
    assert (got[:max(0, adds[0] - lens[0])] == 0).all()


@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 4, 24), (256, 1, 16), (96, 8, 1)])
def test_prompts_under_scales_far_apart(D, group, page):
    lens, adds = [300, 50, 128], [120, 1, 64]
    prompts(21, lens, adds, 1, group, D, page, scale_spread=9).check()
    prompts(22, lens, adds, 1, group, D, page, scales=(2.0 ** -22, 2.0 ** -22)).check()
    a = prompts(23, lens, adds, 1, group, D, page)
    for side in (a.k, a.v):
        side[1][:, ::2] = 0.0  # pages of zeros
    a.d[2].copy_(to_dev(a.k[1])), a.d[4].copy_(to_dev(a.v[1]))
    a.check()


def test_prompts_of_peaked_and_flat_scores():
    prompts(32, [700, 90], [40, 70], 1, 4, 128, 16, q_scale=30.0).check()
    prompts(33, [700, 90], [40, 70], 1, 4, 128, 16, q_scale=0.0).check()
    prompts(34, [700, 90], [40, 70], 1, 4, 64, 24, q_scale=30.0).check()


@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 4, 24), (256, 1, 16), (96, 8, 1)])
def test_nan_of_one_query_of_a_prompt_stays_its_own(D, group, page):
    a = prompts(41, [200, 90], [44, 40], 2, group, D, page)
    clean = host(a.run()).copy()
    q = a.q.copy()
    q[0, 1, 5] = np.nan
    a.d[0].copy_(to_dev(q).view(-1))
    got = host(a.run()).view(np.float16).reshape(a.before.shape)
    assert np.isnan(got[0, 1]).all()
    keep = np.ones(got.shape[:2], bool)
    keep[0, 1] = False
    assert np.array_equal(got[keep].view(np.uint16), clean.view(np.uint16).reshape(got.shape)[keep])


@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 7, 24), (256, 2, 64), (96, 16, 16), (128, 8, 1), (96, 5, 7), (256, 3, 24)])
@pytest.mark.parametrize("causal", [True, False])
def test_nan_codes_of_prompts_reach_only_the_rows_that_see_them(D, group, page, causal):
    lens, adds = [150, 300, 90], [145, 150, 90]
    a = prompts(D + group, lens, adds, 1, group, D, page, causal=causal)
    rng = np.random.default_rng(7)
    for s, (n, m) in enumerate(zip(lens, adds)):
        if s < 2 or causal:  # (without a mask all rows see what the third sequence has: it keeps none)
            for back in (1, 2, m // 2, m - 1):
                t = n - back
                a.v[0].reshape(-1, D)[a.bt[s, t // page] * page + t % page, rng.integers(0, D, 2)] = [0x7F, 0xFF]
    a.k[0].reshape(-1, D)[a.bt[1, 298 // page] * page + 298 % page, 3] = 0x7F
    a.d[1].copy_(to_dev(a.k[0]).view(a.d[1].shape)), a.d[3].copy_(to_dev(a.v[0]).view(a.d[3].shape))
    check_nan(a)


def test_prompts_strides_and_bounds():
    for stride in (1000, 1001):                          # rows at odd addresses
        got = prompts(8, [100, 260], [80, 40], 2, 2, 128, 16, stride=stride).check()
        assert (got[120:] == 7.0).all()
    prompts(9, [100, 260], [80, 40], 2, 2, 128, 16, max_len=5000, max_q=1000).check()
    # lengths past the bound of the call are cut
    a = prompts(12, [100, 260], [80, 40], 2, 2, 128, 16, max_len=128)
    out = a.run()
    a.lens = np.array([100, 128])
    got = host(out).view(np.float16).reshape(a.before.shape).astype(np.float64)
    want, tol = a.want()
    assert (np.abs(got - want)[:80] <= tol[:80]).all()
    a.args = (*a.args[:4], False)                       # (the second one's queries lie past what is kept: they see all of it)
    want, tol = a.want()
    assert (np.abs(got - want)[80:120] <= tol[80:120]).all()


@pytest.mark.parametrize("D, group, page", [(128, 4, 16), (64, 7, 24), (256, 1, 64), (96, 3, 7), (64, 4, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_in_splits(D, group, page, causal):
    """One tile of rows behind many positions, and shorter sequences next to it whose last splits have nothing."""
    a = prompts(D + page, [6000, 300, 1400], [1 + 100 // group, 34, 40], 1, group, D, page, causal=causal)
    assert a.plan[3] > 1
    a.check()


@pytest.mark.parametrize("D, group, page", [(128, 8, 16), (64, 8, 24), (96, 2, 3), (256, 4, 16)])
def test_the_same_rows_by_either_kernel(D, group, page):
    """A call that the kernel for few rows takes, and one with more places whose prompt is the other's."""
    lens, adds = [400, 200], [60, 21]
    a, b = Attn(71, lens, adds, 1, group, D, page), prompts(71, lens, adds, 1, group, D, page)
    plan = w4amd.capi().attention_f8_pages_plan_for(a.view, a.batch, group)
    assert plan[0] == 1 and b.plan[0] >= 3
    assert all(np.array_equal(x, y) for x, y in ((a.bt, b.bt), (a.k[0], b.k[0]), (a.v[0], b.v[0]), (a.q, b.q[:81])))
    a.check(), b.check()


@pytest.mark.parametrize("page", [64, 24])
def test_prompts_on_pages_past_32_bits(page):
    """A pool of more than 2^32 bytes a side: the bytes of the call over a small one."""
    c = w4amd.capi()
    H, group, D = 2, 2, 128
    a = prompts(page, [300, 700], [90, 64], H, group, D, page)
    want = a.run()
    a.check(want)
    npages = 300_000 * 64 // page
    pools = []
    for small in a.d[1:5]:
        big = torch.zeros(H, npages, *small.shape[2:], dtype=small.dtype, device=DEV)
        big[:, npages - a.npages:] = small.flip(1)
        pools.append(big)
    assert pools[0][0].numel() > 1 << 31 and pools[0].numel() > 1 << 32
    a.view = c.f8_pages_view(H, D, page, npages, *[ptr(t) for t in pools])
    a.d[5].copy_(i32(npages - 1 - a.bt))
    assert np.array_equal(host(a.run()), host(want))


def test_prompts_of_every_kind_in_one_workspace():
    kinds = [([3000, 40], [64, 1], 2, 4, 128, 16), ([900, 800], [200, 1], 1, 4, 128, 24), ([5000], [40], 1, 7, 64, 24),
             ([400] * 70, [1] * 69 + [50], 1, 1, 96, 16), ([700, 2000], [40, 33], 1, 2, 256, 64)]
    calls = [prompts(80 + i, *k) for i, k in enumerate(kinds)]
    calls += [Attn(90, [3000, 40], [1, 1], 2, 4, 128, 16), Attn(91, [900], [40], 1, 4, 40, 16)]
    want = [host(x.run()).copy() for x in calls]
    space = torch.zeros(max(x.n for x in calls) + 16, dtype=torch.uint8, device=DEV)
    order = np.random.default_rng(1).integers(0, len(calls), 60)
    outs = [calls[i].run(space=space) for i in order]
    assert all(np.array_equal(host(o), want[i]) for o, i in zip(outs, order))
    for x in calls:
        x.check()


# ---- a step whose bounds are a serving loop's ------------------------------------------------


@pytest.mark.parametrize("group, page, kind", [(4, 16, 4), (4, 24, 3), (20, 16, 3)])
def test_a_captured_step_of_prompts_and_tokens_replayed(group, page, kind):
    """Bounds past what the kernel for few rows takes: prompts, chunks and single tokens under one graph."""
    s = Step(73, 4, 1, group, 128, page, 80, 640 // page, 2300, 300)
    assert w4amd.capi().attention_f8_pages_plan_for(s.view, s.batch, group)[0] == kind
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.launch(side.cuda_stream)

    def replay():
        graph.replay()
        torch.cuda.synchronize()

    for added in ([150, 3, 1, 0], [1, 1, 1, 1], [40, 60, 0, 100], [1, 1, 1, 1], [100, 1, 9, 2]):
        assert s.step(np.array(added), replay)[1] == 0
        torch.ones(1000, device=DEV).sum().item()  # the program's own work between replays
    s.step(np.array([1, 40, 1, 1]), s.launch)


# ---- where things lie ------------------------------------------------------------------------


@pytest.mark.parametrize("adds", [[1, 1], [5, 2], [80, 40]])
@pytest.mark.parametrize("off", [4, 8])
@pytest.mark.parametrize("D", [64, 128])
def test_pools_that_are_not_16_byte_aligned(D, off, adds):
    """Nothing but the vector kernel takes these; head dimensions are the matrix cores'."""
    a = Attn(D + off, [300, 90], adds, 2, 4, D, 16)
    c = w4amd.capi()
    moved = []
    for t in (a.d[1], a.d[3]):
        buf = torch.empty(t.numel() + 16, dtype=torch.uint8, device=DEV)
        moved.append(buf[off:off + t.numel()])
        moved[-1].copy_(t.reshape(-1))
    a.view = c.f8_pages_view(2, D, 16, a.npages, ptr(moved[0]), ptr(a.d[2]), ptr(moved[1]), ptr(a.d[4]))
    assert c.attention_f8_pages_plan_for(a.view, a.batch, 4)[0] == 0
    a.n = c.attention_f8_pages_workspace(a.view, a.batch, 4)
    a.space = torch.zeros(a.n + 16, dtype=torch.uint8, device=DEV)
    a.check()


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("adds", [[1, 1], [70, 40]])
def test_offsets_that_do_not_begin_at_0(D, adds):
    """Packed tokens ahead of the first sequence's are no query, and their rows of `out` stay as they are."""
    before = 9
    a = (prompts if max(adds) > 1 and D != 80 else Attn)(D, [200, 90], adds, 2, 4, D, 16)
    plain = host(a.run()).copy()
    T = len(a.q)
    q = torch.zeros((T + before) * a.row, dtype=torch.int16, device=DEV)
    q[before * a.row:] = a.d[0].view(torch.int16).reshape(-1)
    out = to_dev(np.full((T + before, *a.before.shape[1:]), 7.0, np.float16))
    cu = i32(a.cu + before)
    c = w4amd.capi()
    batch = c.paged_batch(2, T + before, int(max(adds)), 200, ptr(a.d[5]), a.bt.shape[1], ptr(a.d[6]), ptr(cu))
    n = c.attention_f8_pages_workspace(a.view, batch, 4)
    space = torch.zeros(n + 16, dtype=torch.uint8, device=DEV)
    c.attention_f8_pages(a.view, batch, 4, 1, ptr(q), 0, ptr(out), ptr(space), n)
    got = host(out).view(np.float16)
    assert (got[:before] == 7.0).all()
    a.check(out[before:])
    assert np.array_equal(got[before:].reshape(-1).view(np.int16), plain.reshape(-1))


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("adds", [[1, 1, 1, 1], [5, 4, 6, 3], [60, 40, 50, 45]])
def test_offsets_past_the_places(D, adds):
    """More tokens than places: sequences that fit are computed, and nothing is written behind the places."""
    a = (prompts if max(adds) > 8 and D != 80 else Attn)(D, [200, 90, 120, 60], adds, 1, 4, D, 16)
    fit = int(a.cu[2])
    want, tol = (x[:fit] for x in a.want())
    c = w4amd.capi()
    for tokens in (fit, fit + (adds[2] + 1) // 2):
        for max_len in (200, 1000):
            batch = c.paged_batch(4, tokens, int(max(adds)), max_len, ptr(a.d[5]), a.bt.shape[1], ptr(a.d[6]), ptr(a.cu_d))
            n = c.attention_f8_pages_workspace(a.view, batch, 4)
            space, out = torch.zeros(n + 16, dtype=torch.uint8, device=DEV), to_dev(a.before)
            c.attention_f8_pages(a.view, batch, 4, 1, ptr(a.d[0]), 0, ptr(out), ptr(space), n)
            got = host(out).view(np.float16).reshape(a.before.shape).astype(np.float64)
            assert (np.abs(got[:fit] - want) <= tol).all() and (got[tokens:] == 7.0).all()
