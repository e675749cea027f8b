"""A feed-forward block of experts as a serving step runs it: the norm ahead, the router's product, routing, the experts'
products and the way back into the residual stream, next to the library's own GEMM for the shared part; eager and captured."""
import numpy as np
import pytest
import torch

import experts_ref
import w4amd
from devutil import DEV, ptr, to_dev

pytestmark = pytest.mark.gpu


class Block:
    """D wide, E experts of width I, k chosen, one shared expert's way down as a plain packed matrix."""

    def __init__(self, seed, places, D=256, E=8, I=64, k=2, fmt=0):
        c = w4amd.capi()
        rng = np.random.default_rng(seed)
        self.c, self.D, self.E, self.I, self.k, self.places = c, D, E, I, k, places
        self.up, self.down = experts_ref.Experts(rng, E, 2 * I, D, fmt, 64), experts_ref.Experts(rng, E, D, I, 2)
        self.shared = experts_ref.Experts(rng, 1, D, D, 0, 64)
        self.router_w = (rng.normal(size=(E, D)) / np.sqrt(D)).astype(np.float16)
        self.bias = (0.1 * rng.normal(size=E)).astype(np.float32)
        self.pre, self.post = (1 + 0.2 * rng.normal(size=(2, D))).astype(np.float16)
        self.keep = {}

        def dev(name, a):
            self.keep[name] = to_dev(a)
            return ptr(self.keep[name])

        m = self.up
        if fmt == 2:
            self.up_view, self.up_call = c.packed_mx_view(E * 2 * I, D, m.G, dev("uq", m.q), dev("us", m.scales)), c.gemm_experts_mx
        else:
            z = 0 if m.zeros is None else dev("uz", m.zeros)
            self.up_view = c.packed_view(E * 2 * I, D, 64, m.G, fmt == 0, dev("uq", m.q), dev("us", m.scales), z)
            self.up_call = c.gemm_experts
        m = self.down
        self.down_view = c.packed_mx_view(E * D, I, m.G, dev("dq", m.q), dev("ds", m.scales))
        m = self.shared
        self.shared_view = c.packed_view(D, D, 64, m.G, 1, dev("sq", m.q), dev("ss", m.scales))
        self.at = {n: dev(n, a) for n, a in (("router_w", self.router_w), ("bias", self.bias), ("pre", self.pre), ("post", self.post))}
        P = places * k
        for n, shape, t in (("r", (places, D), torch.float32), ("b", (places, D), torch.float16), ("h", (places, D), torch.float16),
                            ("logits", (places, E), torch.float16), ("ids", (places, k), torch.int32),
                            ("w", (places, k), torch.float32), ("order", (P,), torch.int32), ("offsets", (E + 1,), torch.int32),
                            ("mid", (P, I), torch.float16), ("y", (P, D), torch.float16), ("sh", (places, D), torch.float16),
                            ("r2", (places, D), torch.float32), ("h2", (places, D), torch.float16), ("count", (1,), torch.int32)):
            self.keep[n] = torch.zeros(shape, dtype=t, device=DEV)
            self.at[n] = ptr(self.keep[n])
        self.keep["y"].fill_(float("nan"))  # (rows of tokens that are not there are never read)
        self.router = c.router(E, k, score=1, scale=2.0, bias=self.at["bias"])
        self.n = c.route_experts_workspace(self.router, places)
        self.space = torch.zeros(self.n + 16, dtype=torch.uint8, device=DEV)
        self.rows = c.expert_rows(E, places, k, self.at["offsets"], self.at["order"])
        self.first = c.block_norm(D, pre=self.at["pre"])
        self.last = c.block_norm(D, residual_scale=0.5, post=self.at["post"], pre=self.at["pre"])

    def step(self, s):
        c, at, T = self.c, self.at, self.places
        c.residual_norm(self.first, T, 1, at["b"], 0, 0, at["r"], 1, at["r"], at["h"], s)  # in place: b is what came before
        c.gemm_fp16(at["router_w"], at["h"], at["logits"], T, self.E, self.D, s)
        c.route_experts(self.router, at["logits"], 0, 0, T, at["count"], at["ids"], at["w"], at["order"], at["offsets"],
                        ptr(self.space) if self.n else 0, self.n, s)
        self.up_call(self.up_view, self.rows, 1, at["h"], 1, at["mid"], 0, s)
        c.gemm_experts_mx(self.down_view, self.rows, 0, at["mid"], 0, at["y"], 1, s)
        c.gemm(self.shared_view, at["h"], at["sh"], T, s)
        c.residual_norm(self.last, T, self.k, at["y"], at["w"], at["sh"], at["r"], 1, at["r2"], at["h2"], s)

    def fill(self, seed, count):
        rng = np.random.default_rng(seed)
        self.count = count
        self.r0 = rng.normal(size=(self.places, self.D)).astype(np.float32)
        self.b0 = rng.normal(size=(self.places, self.D)).astype(np.float16)
        self.keep["r"].copy_(to_dev(self.r0))
        self.keep["b"].copy_(to_dev(self.b0.view(np.int16)).view(torch.float16))
        self.keep["count"].fill_(count)
        torch.cuda.synchronize()

    def host(self, name):
        torch.cuda.synchronize()
        return self.keep[name].cpu().numpy()

    def check(self):
        """Each operator's result from what the one before it left."""
        T, k, n = self.places, self.k, self.count
        pre = self.pre
        r, off, h, err = experts_ref.residual_norm(self.b0[:, None], None, None, self.r0, None, None, None, pre, None, False, 1e-6, 1.0)
        assert (np.abs(self.host("r") - r) <= experts_ref.rounded(r, off, True)).all()
        assert (np.abs(self.host("h").astype(np.float64) - h) <= experts_ref.rounded(h, err)).all()
        ids, w, bound, order, offsets = experts_ref.route(self.host("logits"), k, sigmoid=True, scale=2.0, bias=self.bias, count=n)
        assert np.array_equal(self.host("ids"), ids) and np.array_equal(self.host("order"), order)
        assert np.array_equal(self.host("offsets"), offsets) and (np.abs(self.host("w") - w) <= bound).all()
        x, mid = self.host("h"), self.host("mid")
        P = offsets[-1]
        want, bound = experts_ref.gemm_experts(self.up, x, order, offsets, k, 1, True, False, np.zeros((T * k, self.I)))
        assert (np.abs(mid.astype(np.float64) - want) <= bound)[:P].all()
        want, bound = experts_ref.gemm_experts(self.down, mid, order, offsets, k, 0, False, True, np.zeros((T * k, self.D)))
        y = self.host("y")
        assert (np.abs(y.astype(np.float64) - want) <= bound)[:n * k].all()
        r, off, h, err = experts_ref.residual_norm(y.reshape(T, k, -1), self.host("w"), self.host("sh"), self.host("r"), self.post, None,
                                                   None, pre, None, False, 1e-6, 0.5)
        assert (np.abs(self.host("r2") - r) <= experts_ref.rounded(r, off, True)).all()
        assert (np.abs(self.host("h2").astype(np.float64) - h) <= experts_ref.rounded(h, err)).all()
        assert np.isfinite(self.host("h2").astype(np.float64)).all()
        # the block as a whole, without roundings between its operators: FP16 in four places one after the other, each
        # half a step of 2^-11 relative to its row, which the gate's slope and the norms carry on: within 2^-7 of the rows' size
        full = self.whole()[:n]
        got = self.host("r2")[:n]
        assert np.linalg.norm(got - full) <= 2.0 ** -7 * np.linalg.norm(full)

    def whole(self):
        T, k, f = self.places, self.k, np.float64
        r = self.r0.astype(f) + self.b0

        def rms(v):
            return v / np.sqrt((v * v).mean(axis=1, keepdims=True) + 1e-6)

        h = rms(r) * self.pre
        ids, w = self.host("ids"), self.host("w")  # (a choice next to a border may go either way)
        up = self.up.w.astype(f).reshape(self.E, 2 * self.I, self.D)
        down = self.down.w.astype(f).reshape(self.E, self.D, self.I)
        b = h @ self.shared.w.astype(f).T
        for t in range(self.count):
            for j in range(k):
                g = up[ids[t, j]] @ h[t]
                b[t] += w[t, j] * (down[ids[t, j]] @ (experts_ref.act(1, g[:self.I]) * g[self.I:]))
        return r + 0.5 * rms(b) * self.post


@pytest.mark.parametrize("places,E,k", [(1, 8, 2), (7, 8, 2), (64, 16, 4), (300, 8, 2)])
@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_a_block_eager(places, E, k, fmt):
    b = Block(places + E, places, E=E, k=k, fmt=fmt)
    for seed in range(2):
        b.fill(seed, places)
        b.step(0)
        b.check()


@pytest.mark.parametrize("places", [4, 48, 320])
def test_a_captured_block_serves_fewer_tokens_too(places):
    """Captured once, replayed with other tokens and fewer of them; eager work of another block in between."""
    b, other = Block(1, places), Block(2, places + 5, E=16, k=3)
    b.fill(0, places)
    b.step(0)
    b.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        b.step(torch.cuda.current_stream().cuda_stream)
    for seed, count in ((1, places), (2, max(1, places // 3)), (3, places - 1), (4, places)):
        b.fill(seed, count)
        graph.replay()
        b.check()
        other.fill(seed, places)
        other.step(0)
        other.check()


def test_a_block_through_the_cpp_api():
    from test_cpp_gates import _run
    assert " 0 failures" in _run("test_experts", 100)
