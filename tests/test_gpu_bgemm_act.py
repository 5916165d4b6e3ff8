"""The BF16 GEMM with bias, activation and residual in its epilogue and its backward product
(bgemm_act.hip) against the formulas in 64 bits.

Tolerances count roundings: a sum of K products, each exact in fp32, is off by at most K 2^-24 of the sum
of their magnitudes in any order; an activation passes on at most 1.13 of that (GELU's largest slope)
and adds the errors of its exponential and reciprocal (16 steps of 2^-24 of |z| + 1 are ample); bf16
outputs are rounded once, by half a step, 2^-8 relative. Column sums add the errors of their rows and
a chain of at most 48 + M / 128 additions."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
ULP, HALF_STEP = 2.0 ** -24, 2.0 ** -8
ACTS = ("none", "relu", "gelu", "silu")
GELU = (0.7978845608028654, 0.044715)


def say(*a):
    print(*a, flush=True)


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(GELU[0] * (z + GELU[1] * z ** 3)))
    return z * torch.sigmoid(z) if name == "silu" else z


def _slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        t = torch.tanh(GELU[0] * (z + GELU[1] * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * GELU[0] * (1 + 3 * GELU[1] * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def _mm(a, b, ta, tb):
    """op(a) op(b) of fp64 matrices or batches of them."""
    a = a.transpose(-1, -2).contiguous() if ta else a
    b = b.transpose(-1, -2).contiguous() if tb else b
    return torch.matmul(a, b)


def _close(got, want, tol, what):
    err = (got.double() - want).abs()
    t = tol + (want.abs() * HALF_STEP if got.dtype == BF else 0) + 1e-37
    assert bool((err <= t).all()), (what, float((err / t).max()), int((err > t).sum()))


class Data:
    """Operands of one product; pad: elements behind every row of every matrix, off: the matrices' first
    element (alignment), batch: None for plain matrices."""

    def __init__(self, M, N, K, ta, tb, seed, batch=None, pad=0, off=0, bias_batch=False):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.M, self.N, self.K, self.ta, self.tb, self.batch = M, N, K, ta, tb, batch
        n = batch or 1

        def mat(rows, cols, std=1.0):
            buf = torch.full((off + n * (rows * (cols + pad) + pad) + 64,), 9.0, device=DEV, dtype=BF)
            v = buf[off:].as_strided((n, rows, cols), (rows * (cols + pad) + pad, cols + pad, 1))
            v.copy_(torch.randn(n, rows, cols, generator=g, device=DEV) * std)
            return buf, (v if batch else v[0])
        self.bufA, self.a = mat(*((K, M) if ta else (M, K)))
        self.bufB, self.b = mat(*((N, K) if tb else (K, N)), std=max(K, 1) ** -0.5)
        self.bufC, self.c = mat(M, N)
        self.bufZ, self.z = mat(M, N)
        self.bufR, self.r = mat(M, N)
        shape = (n, N) if bias_batch else (N,)
        self.bias = torch.randn(*shape, generator=g, device=DEV).to(BF)
        a, b = self.a.double(), self.b.double()
        self.prod = _mm(a, b, ta, tb)
        self.mag = _mm(a.abs(), b.abs(), ta, tb)

    def check_forward(self, hk, act, bias=True, residual=True, preact=True, alpha=1.0, inplace=False):
        bias_t = self.bias if bias else None
        bd = 0.0 if not bias else (self.bias.double()[:, None] if self.bias.dim() == 2 and self.batch
                                   else self.bias.double())
        z = alpha * self.prod + bd
        tz = (self.K + 4) * ULP * (abs(alpha) * self.mag + (bd.abs() if bias else 0.0))
        r = self.r.double() if residual else 0.0
        want = _act(z, act) + r
        tol = 1.13 * tz + 16 * ULP * (z.abs() + 1) + ULP * want.abs()
        out = self.c
        res = self.r if residual else None
        if inplace:
            out.copy_(self.r)
            res = out
        got = hk.bgemm_act(self.a, self.b, bias=bias_t, activation=act, residual=res,
                           preact=self.z if preact else None, out=out, trans_a=bool(self.ta),
                           trans_b=bool(self.tb), alpha=alpha)
        assert got is out
        _close(out, want, tol, f"C {act}")
        if preact:
            _close(self.z, z, tz, f"preact {act}")
        return out.clone()

    def check_backward(self, hk, act, alpha=1.0, shared=True, accumulate=True):
        n = self.batch or 1
        z = self.z.double()
        s = _slope(z, act)
        d = alpha * self.prod * s
        tol = (self.K + 4) * ULP * abs(alpha) * self.mag * s.abs() + (
            16 * ULP * (1 + z.abs()) * (alpha * self.prod).abs())
        db = torch.full((self.N,) if shared else (n, self.N), 0.5, device=DEV)
        out = hk.bgemm_act_backward(self.a, self.b, preact=None if act == "none" else self.z,
                                    activation=act, dbias=db, out=self.c, trans_a=bool(self.ta),
                                    trans_b=bool(self.tb), alpha=alpha, accumulate=accumulate)
        _close(out, d, tol, f"d {act}")
        dims = (0,) if self.batch is None else (0, 1) if shared else (1,)
        want = d.sum(dims)
        rows = self.M * (n if shared else 1)
        tdb = tol.sum(dims) + (48 + rows / 128) * ULP * d.abs().sum(dims)
        if self.batch is None and not shared:
            want, tdb = want[None], tdb[None]
        add = 0.5 if accumulate else 0.0
        _close(db, want + add, tdb + ULP * (want.abs() + 1), f"dbias {act}")
        return out.clone(), db

    def untouched(self):
        """Nothing behind the rows of the outputs was written."""
        for buf, t in ((self.bufC, self.c), (self.bufZ, self.z)):
            t.fill_(9.0)
            assert bool((buf == 9.0).all())


LAYOUTS = [(0, 0), (0, 1), (1, 0), (1, 1)]
SMALL = [(8, 8, 8), (64, 64, 64), (65, 63, 65), (63, 65, 127), (9, 200, 129), (200, 9, 321),
         (127, 129, 191), (333, 77, 1111), (2, 1000, 40), (500, 1, 77), (3, 5, 3), (1, 1, 1),
         (1, 520, 129), (1, 1000, 1024), (1, 77, 5000), (1, 39, 9001), (1, 2000, 9001), (1, 31, 7),
         (17, 136, 1), (130, 264, 72)]


@pytest.mark.parametrize("ta,tb", LAYOUTS)
@pytest.mark.parametrize("M,N,K", SMALL)
def test_small_and_ragged(hk, M, N, K, ta, tb):
    say("act", M, N, K, ta, tb)
    d = Data(M, N, K, ta, tb, 100 + M + N)
    for act in ACTS:
        d.check_forward(hk, act)
        d.check_backward(hk, act)


@pytest.mark.parametrize("ta,tb", LAYOUTS)
@pytest.mark.parametrize("pad,off", [(3, 1), (8, 8), (8, 4), (0, 1)])
@pytest.mark.parametrize("M,N,K", [(96, 200, 136), (1, 264, 512), (70, 65, 33)])
def test_strides_and_alignment(hk, M, N, K, ta, tb, pad, off):
    say("act views", M, N, K, ta, tb, pad, off)
    d = Data(M, N, K, ta, tb, 300 + M, pad=pad, off=off)
    d.check_forward(hk, "gelu", alpha=-0.5)
    d.check_forward(hk, "silu", inplace=True)
    d.check_backward(hk, "gelu", alpha=-0.5)
    d.untouched()


# One product for each way of the planner: (tile rows, splits, columns of the 256-wide tiles)
PLANS = [(512, 768, 2304, 0, 1, 64, False, None), (512, 2304, 768, 0, 0, 128, False, None),
         (2048, 2048, 512, 0, 1, 128, False, None), (192, 384, 4096, 0, 0, 64, True, None),
         (500, 1003, 333, 1, 0, 64, False, None), (300, 299, 4001, 0, 0, 64, True, None),
         (2047, 2049, 257, 0, 1, 128, False, None), (257, 511, 9001, 1, 1, None, True, None),
         (4095, 4097, 65, 1, 0, None, False, None),
         (8192, 1280, 448, 0, 1, 0, False, 160), (8192, 5120, 128, 0, 0, 0, False, 256),
         (4096, 4096, 1024, 1, 0, 0, False, 256), (5208, 6880, 80, 0, 1, 0, False, 256),
         (8192, 1280, 5120, 0, 0, 0, False, 256)]


@pytest.mark.parametrize("M,N,K,ta,tb,tile,split,cols", PLANS)
def test_every_plan(hk, M, N, K, ta, tb, tile, split, cols):
    lib = hk.lib()
    rows, used = (lib.hk_bgemm_small_tile(ta, tb, M, N, K, 1, 0),
                  lib.hk_bgemm_split_count(ta, tb, M, N, K, 1, 0))
    say("act plan", M, N, K, ta, tb, "tile", rows, "splits", used,
        lib.hk_bgemm_tile_rows(ta, tb, M, N, K, 1, 0), lib.hk_bgemm_tile_cols(ta, tb, M, N, K, 1, 0))
    assert rows == tile if tile is not None else rows > 0
    assert (used > 1) == split
    assert cols is None or lib.hk_bgemm_tile_cols(ta, tb, M, N, K, 1, 0) == cols
    d = Data(M, N, K, ta, tb, 500 + M)
    first = d.check_forward(hk, "gelu")
    assert torch.equal(first, d.check_forward(hk, "gelu"))
    d.check_forward(hk, "none", bias=False, preact=False, residual=True, inplace=True)
    d.check_forward(hk, "relu", bias=True, preact=False, residual=False)
    one = d.check_backward(hk, "gelu")
    two = d.check_backward(hk, "gelu")
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    d.check_backward(hk, "relu", accumulate=False)


def test_192_row_tiles(hk):
    lib = hk.lib()
    shape = next((M, 1280, 2560) for M in range(7680, 9000, 192)
                 if lib.hk_bgemm_small_tile(0, 0, M, 1280, 2560, 1, 0) == 0
                 and lib.hk_bgemm_tile_rows(0, 0, M, 1280, 2560, 1, 0) == 192
                 and lib.hk_bgemm_split_count(0, 0, M, 1280, 2560, 1, 0) == 1)
    say("act 192 rows", shape)
    d = Data(*shape, 0, 0, 7)
    d.check_forward(hk, "silu")
    d.check_backward(hk, "silu")


@pytest.mark.parametrize("M,N,K,ta,tb", [(4096, 1272, 1288, 0, 1), (8192, 1280, 512, 0, 1)])
def test_wide_tiles_with_unaligned_outputs(hk, M, N, K, ta, tb):
    """A and B in whole vectors, C, z and the residual not: the 256-wide tiles' element stores."""
    d = Data(M, N, K, ta, tb, 9)
    e = Data(M, N, 8, ta, tb, 10, pad=1, off=1)
    d.bufC, d.c, d.bufZ, d.z, d.bufR, d.r = e.bufC, e.c, e.bufZ, e.z, e.bufR, e.r
    d.check_forward(hk, "gelu")
    d.check_backward(hk, "gelu")
    d.untouched()


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("M,N,K,ta,tb,pad", [(65, 72, 64, 0, 0, 0), (40, 33, 47, 1, 1, 1),
                                             (1, 264, 1024, 0, 1, 0), (300, 304, 4096, 0, 0, 0),
                                             (256, 512, 128, 1, 0, 8)])
@pytest.mark.parametrize("own_bias", [False, True])
def test_batches(hk, batch, M, N, K, ta, tb, pad, own_bias):
    say("act batch", batch, M, N, K, ta, tb, pad, own_bias)
    d = Data(M, N, K, ta, tb, 700 + M, batch=batch, pad=pad, bias_batch=own_bias)
    d.check_forward(hk, "gelu")
    d.check_backward(hk, "gelu", shared=not own_bias)
    d.check_backward(hk, "silu", shared=not own_bias, accumulate=False)
    d.untouched()


@pytest.mark.parametrize("N,K,tb,batch", [(300, 1536, 0, None), (300, 1537, 0, None), (64, 20481, 0, None),
                                          (4001, 3001, 0, None), (14400, 1700, 0, None),
                                          (33001, 300, 0, None), (1500, 2000, 0, 3), (77, 12000, 0, 5),
                                          (1280, 2049, 1, None), (9001, 2100, 1, None), (700, 6000, 1, 3),
                                          (100, 9000, 1, None), (33, 30001, 1, 3)])
def test_every_form_of_one_row(hk, N, K, tb, batch):
    """Whole columns on each workgroup, and k cut into shares."""
    say("act row", N, K, tb, batch)
    d = Data(1, N, K, 0, tb, 900 + N, batch=batch, bias_batch=batch is not None)
    d.check_forward(hk, "gelu")
    d.check_forward(hk, "silu", inplace=True, alpha=0.5)
    d.check_backward(hk, "gelu", shared=batch is None)
    if batch:
        d.check_backward(hk, "gelu")
    d.untouched()


@pytest.mark.parametrize("M,N,K,tb", [(512, 768, 2304, 1), (512, 2304, 768, 0), (300, 304, 4096, 0),
                                      (301, 303, 1001, 1), (8192, 1280, 448, 1), (8192, 5120, 128, 0),
                                      (1, 1000, 1024, 0), (1, 1000, 5000, 0), (1, 1000, 5000, 1)])
def test_in_place(hk, M, N, K, tb):
    """The residual and the backward pass's preact as the output, on every kind of plan."""
    say("act in place", M, N, K, tb)
    d = Data(M, N, K, 0, tb, 77 + M)
    kw = dict(trans_b=bool(tb), activation="gelu")
    want = hk.bgemm_act(d.a, d.b, bias=d.bias, residual=d.r, preact=d.z, **kw)
    got = d.r.clone()
    hk.bgemm_act(d.a, d.b, bias=d.bias, residual=got, out=got, **kw)
    assert torch.equal(got, want)
    db = torch.zeros(2, N, device=DEV)
    want = hk.bgemm_act_backward(d.a, d.b, preact=d.z, dbias=db[0], **kw)
    got = d.z.clone()
    hk.bgemm_act_backward(d.a, d.b, preact=got, out=got, dbias=db[1], **kw)
    assert torch.equal(got, want) and torch.equal(db[0], db[1])


def test_leading_dimensions_past_the_tiles(hk):
    """Leading dimensions from 2^22 on run on the plain kernel."""
    M, N, K, ld = 70, 40, 24, (1 << 22) + 8
    big = torch.empty(M * ld, device=DEV, dtype=BF)
    d = Data(M, N, K, 0, 0, 21)
    a = big.as_strided((M, K), (ld, 1))
    a.copy_(d.a)
    d.a = a
    d.check_forward(hk, "gelu")
    d.check_backward(hk, "gelu")


def test_without_k_and_without_rows(hk):
    d = Data(40, 24, 0, 0, 0, 23)
    d.check_forward(hk, "silu")
    d.check_backward(hk, "silu")
    e = torch.empty(0, 24, device=DEV, dtype=BF)
    w = torch.randn(16, 24, device=DEV).to(BF)
    x = torch.empty(0, 16, device=DEV, dtype=BF)
    assert hk.bgemm_act(x, w).shape == (0, 24)
    db = torch.full((24,), 2.0, device=DEV)
    hk.bgemm_act_backward(x, w, preact=e, activation="relu", dbias=db)
    assert bool((db == 2).all())
    hk.bgemm_act_backward(x, w, preact=e, activation="relu", dbias=db, accumulate=False)
    assert bool((db == 0).all())
    assert hk.bgemm_act(torch.ones(3, 0, device=DEV, dtype=BF), torch.ones(0, 0, device=DEV, dtype=BF)).shape == (3, 0)


def test_values_that_are_not_finite(hk):
    """NaN and infinity pass as the formulas have them; the derivative of a large z is 0 or 1."""
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[0.0, -0.0, inf, -inf, nan, 3e38, -3e38, 1e19, -1e19, 100.0, -100.0, 64.0]],
                     device=DEV).to(BF)
    n = z.shape[1]
    ones, eye = torch.ones(2, n, device=DEV, dtype=BF), torch.eye(n, device=DEV).to(BF)
    for rows in (1, 2):
        for act in ("relu", "gelu", "silu"):
            got = hk.bgemm_act_backward(ones[:rows], eye, preact=z.expand(rows, n).contiguous(),
                                        activation=act)
            want = torch.tensor([0.5, 0.5, 1, 0, nan, 1, 0, 1, 0, 1, 0, 1])
            if act == "relu":
                want[:2] = 0
            assert torch.allclose(got[0].float().cpu(), want, rtol=0, atol=0, equal_nan=True), act
        # forward: z = the bias
        zero = torch.zeros(rows, n, device=DEV, dtype=BF)
        for act in ACTS:
            p = torch.empty(rows, n, device=DEV, dtype=BF)
            got = hk.bgemm_act(zero, eye, bias=z[0], activation=act, preact=p)
            assert torch.equal(p[0].nan_to_num(7.0), z[0].nan_to_num(7.0))
            want = _act(z[0].float().cpu(), act)
            pick = torch.isfinite(z[0].float().cpu()) | torch.isnan(z[0].float().cpu())
            assert torch.allclose(got[0].float().cpu()[pick], want[pick].to(BF).float(), rtol=2 ** -7,
                                  atol=1e-30, equal_nan=True), act


def test_two_graphs_captured_on_one_stream(hk):
    """Split products with a bias gradient: every graph has its own workspace, as the eager calls do."""
    s = torch.cuda.Stream()
    sets = []
    for M, N, K in ((192, 384, 4096), (300, 299, 4001), (1, 1000, 9000)):
        d = Data(M, N, K, 0, 0, 31 + M)
        assert M == 1 or hk.lib().hk_bgemm_split_count(0, 0, M, N, K, 1, 0) > 1
        db = torch.zeros(N, device=DEV)
        out, pre = torch.empty_like(d.c), torch.empty_like(d.c)
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            hk.bgemm_act(d.a, d.b, bias=d.bias, activation="gelu", residual=d.r, preact=pre, out=out)
            g = hk.bgemm_act_backward(d.a, d.b, preact=d.z, activation="gelu", dbias=db,
                                      accumulate=False)
        sets.append((graph, d, out, pre, g, db))
    for _ in range(3):
        for graph, d, *_ in sets:
            d.a.mul_(-0.5).add_(0.01)
            graph.replay()
        torch.cuda.synchronize()
        for graph, d, out, pre, g, db in sets:
            p2, db2 = torch.empty_like(pre), torch.zeros_like(db)
            o2 = hk.bgemm_act(d.a, d.b, bias=d.bias, activation="gelu", residual=d.r, preact=p2)
            g2 = hk.bgemm_act_backward(d.a, d.b, preact=d.z, activation="gelu", dbias=db2,
                                       accumulate=False)
            assert torch.equal(out, o2) and torch.equal(pre, p2)
            assert torch.equal(g, g2) and torch.equal(db, db2)


def test_captured_call_without_a_workspace_is_refused(hk):
    d = Data(192, 384, 4096, 0, 0, 41)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    args = lambda ws, n: (0, 0, 192, 384, 4096, 0x3F80, d.a.data_ptr(), 4096, 0, d.b.data_ptr(), 384,  # noqa: E731
                          0, None, 0, 2, None, 0, 0, None, 0, 0, d.c.data_ptr(), 384, 0, 1, ws, n)
    need = hk.lib().hk_bgemm_act_workspace(0, 0, 192, 384, 4096, 1, 0)
    assert need > 0
    with torch.cuda.graph(graph, stream=s):
        status = hk.lib().hk_bgemm_act(*args(None, 0), s.cuda_stream)
        d.c.zero_()
    assert status == 900  # hipErrorStreamCaptureUnsupported
    ws = torch.empty(need, device=DEV, dtype=torch.uint8)
    lib = hk.lib()
    assert lib.hk_bgemm_act(*args(ws.data_ptr(), 256), hk._stream()) == 1
    assert lib.hk_bgemm_act(*args(ws.data_ptr() + 4, need), hk._stream()) == 1
    assert lib.hk_bgemm_act(*args(ws.data_ptr(), need), hk._stream()) == 0
    want = d.check_forward(hk, "gelu", bias=False, residual=False, preact=False)
    assert torch.equal(d.c, want)


def test_calls_on_two_streams_at_once(hk):
    d = [Data(300, 299, 4001, 0, 0, 51 + i) for i in range(2)]
    want = [x.check_backward(hk, "gelu", accumulate=False) for x in d]
    streams = [torch.cuda.Stream() for _ in d]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for x, s in zip(d, streams):
            with torch.cuda.stream(s):
                db = torch.empty(x.N, device=DEV)
                got.append((hk.bgemm_act_backward(x.a, x.b, preact=x.z, activation="gelu", dbias=db,
                                                  accumulate=False), db))
    torch.cuda.synchronize()
    for i, (o, db) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(db, want[i % 2][1])


def test_against_the_separate_kernels(hk):
    """One hidden layer: the product with bias, GELU forward and backward as the library has them."""
    M, I, O = 256, 320, 640
    d = Data(M, O, I, 0, 0, 61)
    pre = torch.empty(M, O, device=DEV, dtype=BF)
    y = hk.bgemm_act(d.a, d.b, bias=d.bias, activation="gelu", preact=pre)
    h = torch.empty(M, O, device=DEV, dtype=BF)
    hk.call("hk_bgemm_addmm", M, O, I, 0x3F80, d.a.data_ptr(), I, 0, d.b.data_ptr(), O, 0, 0x3F80,
            d.bias.data_ptr(), O, h.data_ptr(), O, 0, 1, hk._stream())
    # h and pre round the same sums; the plan of both is the same
    assert torch.equal(pre, h)
    sep = hk.gelu_forward(h)
    # three roundings lie between them: h's, which the slope of at most 1.13 passes on, y's own and
    # sep's own. Either of the last two alone may move a value by half a step, so both count: values
    # in [1, 2) may be one step of 2^-7 apart, 2 * 2^-8.
    tol = (1.13 * h.double().abs() + sep.double().abs() + y.double().abs()) * HALF_STEP + 1e-6
    assert bool(((y.double() - sep.double()).abs() <= tol).all())
