"""Products of pairs' rows with their experts' packed matrices on the GPU, against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import experts_ref
import w4amd
from devutil import DEV, ptr, to_dev

pytestmark = pytest.mark.gpu


def spread(rng, T, k, E, counts=None):
    """(order, offsets): T tokens' k different experts each, or so many pairs of each expert as `counts` says."""
    if counts is None:
        flat = np.stack([rng.permutation(E)[:k] for _ in range(T)]).reshape(-1)
    else:
        flat = rng.permutation(np.repeat(np.arange(E), counts))
        assert len(flat) == T * k
    order = np.argsort(flat, kind="stable").astype(np.int32)
    return order, np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=E))]).astype(np.int32)


class Products:
    def __init__(self, seed, T, k, E, width, K, fmt=0, gs=32, act=1, from_tokens=True, to_pairs=False, counts=None, plan=None,
                 skew=0, slack=0):
        c = w4amd.capi()
        rng = np.random.default_rng(seed)
        self.args = (T, k, E, width, K, act, from_tokens, to_pairs)
        self.m = experts_ref.Experts(rng, E, width * (2 if act else 1), K, fmt, gs)
        self.order, self.offsets = spread(rng, T, k, E, counts) if plan is None else plan
        self.x = rng.normal(size=(T if from_tokens else T * k, K)).astype(np.float16)
        m = self.m

        def put(a):  # `skew` elements behind an aligned address
            flat = np.concatenate([np.zeros(skew, a.dtype), a.reshape(-1), np.zeros(slack, a.dtype)])
            d = to_dev(flat)
            return d, ptr(d) + skew * a.itemsize

        self.keep = [put(a) for a in (m.q, m.scales) + (() if m.zeros is None else (m.zeros,))]
        at = [p for _, p in self.keep]
        self.x_d, self.x_at = put(self.x)
        if fmt == 2:
            self.view, self.fn = c.packed_mx_view(E * m.R, K, m.G, at[0], at[1]), c.gemm_experts_mx
        else:
            self.view, self.fn = c.packed_view(E * m.R, K, gs, m.G, fmt == 0, *at), c.gemm_experts
        self.order_d, self.offsets_d = to_dev(self.order), to_dev(self.offsets)
        self.rows = c.expert_rows(E, T, k, ptr(self.offsets_d), ptr(self.order_d))
        self.before = rng.normal(size=(T * k, width)).astype(np.float16)
        self.out, self.out_at = put(self.before)
        self.skew = skew

    def call(self, stream=0):
        T, k, E, width, K, act, from_tokens, to_pairs = self.args
        self.fn(self.view, self.rows, act, self.x_at, int(from_tokens), self.out_at, int(to_pairs), stream)
        return self

    def got(self):
        torch.cuda.synchronize()
        return self.out.cpu().numpy().view(np.float16)[self.skew:self.skew + self.before.size].reshape(self.before.shape)

    def check(self):
        T, k, E, width, K, act, from_tokens, to_pairs = self.args
        got = self.got()
        want, bound = experts_ref.gemm_experts(self.m, self.x, self.order, self.offsets, k, act, from_tokens, to_pairs, self.before)
        off = np.abs(got.astype(np.float64) - want)
        assert (off <= bound).all(), (float(np.nanmax(off - bound)), np.argwhere(~(off <= bound))[:5])
        done = bound > 0
        rel = np.sqrt((off[done] ** 2).sum() / max((want[done] ** 2).sum(), 1e-300))
        assert rel <= 1e-3, rel  # (the library's gate of a product)
        assert np.array_equal(got[~done], self.before[~done])
        return self


SHAPES = [(fmt, gs) for fmt, sizes in ((0, (32, 64, 128, 8, 24, 48, 256)), (1, (32, 64, 128, 8, 40)), (2, (32,))) for gs in sizes]


@pytest.mark.parametrize("fmt,gs", SHAPES)
@pytest.mark.parametrize("act,from_tokens,to_pairs", [(1, True, False), (0, False, True), (2, False, False), (0, True, True)])
@pytest.mark.parametrize("T,k,E", [(1, 2, 4), (5, 2, 3), (40, 3, 8)])
def test_formats_and_ways(T, k, E, act, from_tokens, to_pairs, fmt, gs):
    Products(gs + T, T, k, E, 64, 256, fmt, gs, act, from_tokens, to_pairs).call().check()


@pytest.mark.parametrize("K", [1, 7, 8, 31, 40, 96, 100, 128, 160, 200, 384, 500, 1056, 2048])
@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_lengths(K, fmt):
    Products(K, 9, 2, 3, 48, K, fmt, 32, 1).call().check()
    Products(K + 1, 70, 2, 3, 33, K, fmt, 64, 0, False, True).call().check()


@pytest.mark.parametrize("width", [1, 2, 3, 7, 16, 17, 31, 32, 48, 63, 64, 65, 100, 128, 129, 160, 255, 256, 300])
@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_widths(width, fmt):
    Products(width, 6, 2, 3, width, 256, fmt, 128, 1).call().check()
    Products(width + 1, 6, 2, 3, width, 256, fmt, 64, 0, False, True).call().check()
    Products(width + 2, 150, 2, 3, width, 256, fmt, 32, 1).call().check()
    Products(width + 3, 150, 2, 3, width, 256, fmt, 32, 0, False, True).call().check()


@pytest.mark.parametrize("counts", [[0, 0, 64, 0], [64, 0, 0, 0], [0, 0, 0, 64], [1, 62, 0, 1], [15, 16, 17, 16], [31, 32, 1, 0],
                                    [1, 1, 1, 61], [129, 127, 128, 0], [300, 0, 1, 83], [1000, 3, 17, 4]])
@pytest.mark.parametrize("fmt,act", [(0, 1), (1, 0), (2, 1)])
def test_uneven_experts(counts, fmt, act):
    T = sum(counts)
    for from_tokens, to_pairs in ((True, False), (False, True)):
        Products(T, T, 1, 4, 96, 384, fmt, 64, act, from_tokens, to_pairs, counts=counts).call().check()


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (3, 1, 300), (2, 8, 1024), (30, 6, 65), (260, 4, 4), (700, 2, 129)])
@pytest.mark.parametrize("fmt", [0, 2])
def test_numbers_of_experts(T, k, E, fmt):
    Products(E, T, k, E, 32, 128, fmt, 32, 1).call().check()
    Products(E, T, k, E, 32, 128, fmt, 32, 0, False, True).call().check()


def test_pairs_without_an_expert():
    """Their rows stay as they are; places whose order is no pair are not multiplied."""
    rng = np.random.default_rng(5)
    for T, k, E in ((20, 2, 4), (300, 2, 4)):
        order, offsets = spread(rng, T, k, E)
        last = int(offsets[-2])  # the last expert's pairs are nobody's
        offsets[-1] = last
        order[last:] = -1
        order[3], order[7] = -1, 2 ** 31 - 1
        for act, from_tokens, to_pairs in ((1, True, False), (0, False, True), (0, True, True)):
            Products(T, T, k, E, 64, 256, 0, 64, act, from_tokens, to_pairs, plan=(order, offsets)).call().check()
    none = np.zeros(5, np.int32)
    Products(1, 8, 2, 4, 64, 256, 0, 64, plan=(np.full(16, -1, np.int32), none)).call().check()


def test_one_token_twice_at_one_expert():
    """A plan of the user's own may name an expert several times for a token."""
    flat = np.array([1, 1, 0, 1, 1, 1])
    order = np.argsort(flat, kind="stable").astype(np.int32)
    offsets = np.array([0, 1, 6], np.int32)
    Products(2, 3, 2, 2, 64, 256, 0, 64, plan=(order, offsets)).call().check()
    Products(3, 3, 2, 2, 64, 256, 2, 32, 0, True, True, plan=(order, offsets)).call().check()


@pytest.mark.parametrize("skew", [1, 2, 4, 8])
@pytest.mark.parametrize("fmt,gs", [(0, 128), (0, 64), (0, 32), (1, 64), (1, 128), (1, 32), (2, 32)])
def test_arrays_at_any_address(skew, fmt, gs):
    for T in (6, 90, 400):
        Products(T, T, 2, 4, 64, 256, fmt, gs, 1, skew=skew).call().check()
        Products(T, T, 2, 4, 64, 256, fmt, gs, 0, False, True, skew=skew).call().check()


@pytest.mark.parametrize("fmt,gs", [(0, 128), (1, 128), (1, 64), (2, 32)])
def test_odd_numbers_of_scales(fmt, gs):
    """Arrays of scales that end inside a dword."""
    for T in (6, 90, 400):
        Products(T, T, 1, 3, 35, 128, fmt, gs, 0, False, True).call().check()
        Products(T, T, 1, 3, 35, 384, fmt, gs, 0).call().check()


@pytest.mark.parametrize("T,k,E,width,K,fmt,gs", [(4, 4, 8, 704, 1024, 0, 128), (64, 2, 8, 704, 1024, 1, 64), (33, 4, 8, 512, 1408, 2, 32),
                                                  (512, 2, 8, 512, 1024, 0, 128), (300, 4, 8, 352, 1088, 1, 32),
                                                  (700, 2, 8, 576, 1408, 2, 32)])
def test_larger(T, k, E, width, K, fmt, gs):
    Products(T, T, k, E, width, K, fmt, gs, 1).call().check()
    Products(T + 1, T, k, E, width, K, fmt, gs, 0, False, True).call().check()


@pytest.mark.parametrize("fmt,gs", [(0, 32), (0, 64), (0, 96), (0, 128), (0, 192), (0, 256), (0, 384), (0, 512), (1, 32), (1, 64),
                                    (1, 96), (1, 128), (1, 192), (1, 256), (1, 384), (1, 512), (2, 32)])
@pytest.mark.parametrize("K", [576, 1600, 2112, 3136])
def test_groups_along_a_long_row(K, fmt, gs):
    """Every kernel: a row an expert, some, dozens, hundreds; the last group, chunk, stage and window are cut short."""
    for T in (1, 20, 90, 300):
        Products(K + T, T, 2 if T > 1 else 1, 4, 40, K, fmt, gs, 1).call().check()
        Products(K + T + 1, T, 2 if T > 1 else 1, 3, 35 if K % 128 else 36, K, fmt, gs, 0, False, True).call().check()


@pytest.mark.parametrize("T", [3, 30, 300])
def test_rows_that_are_not_finite_stay_in_their_row(T):
    p = Products(T, T, 2, 4, 64, 256, 0, 64, 0, True, True)
    p.x[1, 5], p.x[2, 7] = np.nan, np.inf
    p.x_d.copy_(to_dev(p.x.reshape(-1)))
    got = p.call().got()
    bad = np.repeat(np.isin(np.arange(T), (1, 2)), 2)
    assert np.isnan(got[2:4]).all() and not np.isfinite(got[4:6]).any()
    assert np.isfinite(got[~bad]).all()


def test_results_past_fp16_are_infinite():
    p = Products(1, 3, 1, 2, 64, 128, 0, 64, 0, True, True)
    p.x[:] = 60000
    p.x_d.copy_(to_dev(p.x.reshape(-1)))
    got = p.call().got().astype(np.float64)
    want, bound = experts_ref.gemm_experts(p.m, p.x, p.order, p.offsets, 1, 0, True, True, p.before)
    sure = np.abs(want) > 65520 + bound
    assert sure.any() and (got[sure] == np.sign(want[sure]) * np.inf).all()


@pytest.mark.parametrize("T", [2, 40, 400])
def test_a_captured_call_is_replayed_on_other_plans(T):
    p = Products(T, T, 2, 8, 64, 256, 0, 64).call().check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        p.call(torch.cuda.current_stream().cuda_stream)
    for seed in range(4):
        rng = np.random.default_rng(seed)
        p.order, p.offsets = spread(rng, T, 2, 8)
        p.order_d.copy_(to_dev(p.order))
        p.offsets_d.copy_(to_dev(p.offsets))
        graph.replay()
        p.check()
        Products(seed, T + 1, 2, 4, 32, 128, 2).call().check()


def test_streams_and_repeated_calls_give_the_same_bytes():
    for T in (3, 50, 500):
        p = Products(T, T, 2, 8, 128, 512, 1, 64)
        first = p.call().got().copy()
        streams = [torch.cuda.Stream() for _ in range(3)]
        for s in streams * 2:
            p.out.zero_()
            torch.cuda.synchronize()
            p.call(s.cuda_stream)
            assert np.array_equal(p.got().view(np.uint16), first.view(np.uint16))


@pytest.mark.parametrize("fmt,gs", [(0, 128), (1, 64), (2, 32)])
def test_codes_past_four_gigabytes(fmt, gs):
    """The last of 40 experts of 67 million weights each, by every kernel; some columns and rows are checked."""
    c = w4amd.capi()
    E, R, K = 40, 16384, 16384
    gen = torch.Generator(device=DEV)
    gen.manual_seed(fmt)
    G = K // (32 if fmt == 2 else gs)
    q = torch.randint(-2 ** 31, 2 ** 31 - 1, (E * R, K // 8), dtype=torch.int32, device=DEV, generator=gen)
    zeros = torch.randint(-2 ** 31, 2 ** 31 - 1, (E * R, (G + 7) // 8), dtype=torch.int32, device=DEV, generator=gen)
    if fmt == 2:
        scales = torch.randint(119, 124, (E * R, G), dtype=torch.uint8, device=DEV, generator=gen)
        view, fn = c.packed_mx_view(E * R, K, G, ptr(q), ptr(scales)), c.gemm_experts_mx
    else:
        scales = (torch.rand(E * R, G, device=DEV, generator=gen) * 0.004 + 0.001).half()
        view = c.packed_view(E * R, K, gs, G, fmt == 0, ptr(q), ptr(scales), ptr(zeros) if fmt else 0)
        fn = c.gemm_experts
    cols = np.array([0, 1, 777, R // 2 - 1])
    rows = (E - 1) * R + np.concatenate([cols, R // 2 + cols])
    words = q[rows].cpu().numpy().view(np.uint32)
    codes = (words[:, :, None] >> (4 * np.arange(8, dtype=np.uint32)) & 15).reshape(len(rows), K).astype(np.int64)
    group = np.arange(K) // (K // G)
    s = scales[rows].cpu().numpy()
    if fmt == 2:
        w = experts_ref.E2M1[codes] * np.exp2(s.astype(np.float64) - 127)[:, group]
    else:
        z = 8
        if fmt:
            zw = zeros[rows].cpu().numpy().view(np.uint32)
            z = (zw[:, :, None] >> (4 * np.arange(8, dtype=np.uint32)) & 15).reshape(len(rows), -1)[:, group].astype(np.int64)
        w = (codes - z) * s.astype(np.float64)[:, group]
    w = w.astype(np.float16).astype(np.float64)
    seen = set()
    for T in (1, 9, 30, 1920):
        seen.add(c.gemm_experts_plan_for(fmt, E, R, K, gs, T, 1))
        x = torch.randn(T, K, device=DEV, generator=gen).half()
        order = torch.arange(T, dtype=torch.int32, device=DEV)
        offsets = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        offsets[E] = T
        out = torch.zeros(T, R // 2, dtype=torch.float16, device=DEV)
        fn(view, c.expert_rows(E, T, 1, ptr(offsets), ptr(order)), 1, ptr(x), 1, ptr(out), 0)
        torch.cuda.synchronize()
        some = np.unique([0, T // 2, T - 1])
        xs = x[some].cpu().numpy().astype(np.float64)
        y, off = xs @ w.T, (K + 8) * experts_ref.U * (np.abs(xs) @ np.abs(w).T)
        a, n = experts_ref.act(1, y[:, :4]), np.abs(y[:, 4:])
        want = a * y[:, 4:]
        err = (1.13 * off[:, :4] + np.abs(a) * (12 + np.abs(y[:, :4])) * 2 * experts_ref.U) * (n + off[:, 4:]) + np.abs(a) * off[:, 4:]
        got = out[some][:, cols].cpu().numpy().astype(np.float64)
        bound = err + (np.abs(want) + err) * experts_ref.H + experts_ref.SUB
        assert (np.abs(got - want) <= bound).all(), (T, float(np.abs(got - want).max()))
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        assert rel <= 1e-3, (T, rel)
    assert seen == {1, 3, 4}
