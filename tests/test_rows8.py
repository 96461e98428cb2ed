"""Products of 8-bit rows (pgan_quant_rows, pgan_gemm_q8, pgan_linear_q8) and the fold of a stride-2 transposed convolution
(pgan_up_fold_q8, pgan_up_fold) against their definitions in 64 bits, and their refusals.

Tolerances: u = 2^-24 is the largest relative error of one fp32 rounding.  The product's sum of whole numbers is exact; its
conversion to fp32, the product of the two scales, their product with the sum and the addition of the bias round once each:
3 u |y - bias| + u |y|, 4 u (|y - bias| + |bias|) is used.  The fold's sum of four taps and a shift takes four additions: at
most 4 u of the sum of their magnitudes.  A result in fewer bits adds half a step of its type."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

U = 2.0 ** -24
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def hip():
    from pgan_hip import HipOps
    return HipOps(torch.device(DEV), ws_floats=4, max_samples=1)


def rnd(rng, *shape, scale=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32))


def half_step(x, dtype):
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
    return torch.finfo(dtype).eps / 2 * x.abs() * (dtype != torch.float32) + least


def lrelu(x):
    return torch.where(x > 0, x, x * 0.1)


def codes_of(x):
    """Codes and scales by their definition, on the CPU in fp32."""
    amax = x.abs().amax(dim=1).clamp_min(2.0 ** -100)
    fine = torch.isfinite(amax)
    inv = torch.full_like(amax, 127.0) / amax
    q = torch.where(fine[:, None], torch.round(x * inv[:, None]), 0.0)
    return q.to(torch.int8), torch.where(fine, amax * torch.tensor(1 / 127, dtype=torch.float32), torch.nan)


def same(a, b):
    assert a.shape == b.shape and torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def rows8(t, fill=85):
    """Codes as a view of a wider buffer: between the rows' ends and the next rows stands `fill`."""
    T, K = t.shape
    buf = torch.full((T + 1, (K + 15) // 16 * 16 + 16), fill, dtype=torch.int8)
    buf[:T, :K] = t
    return buf.to(DEV)[:T, :K]


def rest_kept(view, fill=85):
    base = view._base.clone()
    base[:view.shape[0], :view.shape[1]] = fill
    assert bool((base == fill).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,gap", [(1, 1, 0), (1, 128, 0), (5, 7, 0), (3, 64, 8), (16, 512, 0), (33, 1001, 5), (2, 8192, 0), (130, 256, 16),
                                     (1, 20000, 0), (9, 2056, 0), (1000, 72, 0)])
def test_quant_rows(hip, dtype, T, K, gap):
    rng = np.random.default_rng(T * 1000 + K)
    x = rnd(rng, T, K + gap).to(dtype)
    for neg in (False, True):
        want, ws = codes_of(lrelu(x[:, :K].float()) if neg else x[:, :K].float())
        q = rows8(torch.zeros(T, K, dtype=torch.int8))
        scale = torch.full((T + 3,), 7.0, device=DEV)
        hip.quant_rows(x.to(DEV)[:, :K], q, scale, lrelu=neg)
        assert torch.equal(q.cpu(), want)
        same(scale[:T].cpu(), ws)
        assert bool((scale[T:] == 7).all())
        rest_kept(q)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [40, 512, 3001])
def test_quant_rows_of_odd_values(hip, K):
    """Rows of zeros, of the smallest numbers, of the largest, with infinities and NaN, each beside ordinary rows."""
    rng = np.random.default_rng(4)
    x = rnd(rng, 10, K)
    x[1] = 0
    x[2] *= 1e-38
    x[3] = 1e-45
    x[4] = x[4] / x[4].abs().max() * 3.4028234e38
    x[5, K // 2] = float("inf")
    x[6, K - 1] = float("nan")
    x[7, 0] = float("-inf")
    x[8] = -x[8].abs()
    want, ws = codes_of(x)
    q, scale = rows8(torch.ones(10, K, dtype=torch.int8)), torch.zeros(10, device=DEV)
    hip.quant_rows(x.to(DEV), q, scale)
    assert torch.equal(q.cpu(), want)
    same(scale.cpu(), ws)
    assert bool(torch.isnan(scale.cpu()[5:8]).all()) and bool(torch.isfinite(scale.cpu()[[0, 1, 2, 3, 4, 8, 9]]).all())


SHAPES = [(1, 1, 1), (1, 128, 8192), (1, 4096, 16), (2, 33, 70), (16, 512, 4096), (17, 15, 16), (31, 640, 33), (64, 128, 130), (100, 1001, 257),
          (128, 128, 128), (129, 129, 129), (200, 2048, 64), (300, 64, 16), (777, 1001, 1234), (1024, 64, 16), (4096, 256, 2048),
          (513, 4100, 515), (2, 131072, 20), (4, 8192, 1024), (8, 1000, 5000)]


def product_case(seed, T, K, N):
    rng = np.random.default_rng(seed)
    q = torch.from_numpy(rng.integers(-127, 128, (T, K)).astype(np.int8))
    w = torch.from_numpy(rng.integers(-127, 128, (N, K)).astype(np.int8))
    return q, w, rnd(rng, T).abs() * 0.01 + 1e-4, rnd(rng, N).abs() * 0.01, rnd(rng, N)


def product64(q, qs, w, ws, bias):
    y = (q.double() @ w.double().t()) * (qs.double()[:, None] * ws.double()[None])
    tol = 4 * U * (y.abs() + (0 if bias is None else bias.double().abs()))
    return (y if bias is None else y + bias.double()), tol


def check_product(got, want, tol, dtype):
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol + half_step(want.abs() + tol, dtype))
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outside, worst {float(off.max())}, first {bad.nonzero()[0].tolist()}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,N", SHAPES)
def test_gemm_q8(hip, T, K, N, dtype):
    q, w, qs, ws, bias = product_case(T + K + N, T, K, N)
    want, tol = product64(q, qs, w, ws, bias)
    buf = torch.full((T + 2, N + 8), 7.0, dtype=dtype, device=DEV)        # rows of a wider buffer: what is around stays
    hip.gemm_q8(rows8(q), qs.to(DEV), rows8(w), ws.to(DEV), buf[:T, :N], bias.to(DEV))
    check_product(buf[:T, :N], want, tol, dtype)
    assert bool((buf[T:] == 7).all()) and bool((buf[:, N:] == 7).all())
    y = torch.empty(T, N, dtype=dtype, device=DEV)
    hip.gemm_q8(rows8(q, 3), qs.to(DEV), rows8(w, -9), ws.to(DEV), y)     # without a bias, other bytes between the rows
    want, tol = product64(q, qs, w, ws, None)
    check_product(y, want, tol, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,Ks", [(4097, 4100, (1024, 1030)), (7300, 1025, (512, 1001)), (7300, 2100, (512, 577, 1001)),
                                    (6500, 1300, (1, 64, 65, 128, 190, 200, 256, 500)),
                                    (5000, 1100, (1, 128, 129, 256, 300, 513, 700)), (1000, 700, (1, 127, 129, 300, 385, 2000)), (650, 600, (1, 128, 129, 512, 520, 900)),
                                    (100000, 30, (1, 64, 70, 129, 200)), (9000, 32, (33, 4096))])
def test_gemm_q8_of_every_tile(hip, T, N, Ks):
    """Each tile size with K of one stage of its ring, of a few, of more than it holds, and with a rest.  (The sums of the oracle
    are whole numbers below 2^53: exact on the device too.)"""
    for K in Ks:
        q, w, qs, ws, bias = product_case(T + K + N, T, K, N)
        y = torch.full((T + 1, N), 7.0, dtype=torch.bfloat16, device=DEV)
        hip.gemm_q8(rows8(q, 5), qs.to(DEV), rows8(w, -3), ws.to(DEV), y[:T], bias.to(DEV))
        want, tol = (v.cpu() for v in product64(*(v.to(DEV) for v in (q, qs, w, ws, bias))))
        check_product(y[:T], want, tol, torch.bfloat16)
        assert bool((y[T] == 7).all())


@pytest.mark.gpu
def test_the_sum_is_exact_at_its_largest(hip):
    K = 131072
    q = torch.full((3, K), 127, dtype=torch.int8)
    w = torch.full((40, K), -127, dtype=torch.int8)
    w[1] = 127
    y = torch.empty(3, 40, device=DEV)
    hip.gemm_q8(rows8(q), torch.ones(3, device=DEV), rows8(w), torch.ones(40, device=DEV), y)
    want = torch.full((3, 40), -127.0 * 127 * K)
    want[:, 1] *= -1
    assert torch.equal(y.cpu(), want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("xt", TYPES)
@pytest.mark.parametrize("T,K,N", SHAPES)
def test_linear_q8(hip, T, K, N, xt):
    """The same result as its two halves, bit for bit, and that of the definition."""
    rng = np.random.default_rng(T + 7 * K)
    x = (rnd(rng, T, K + 3) * torch.exp(rnd(rng, T, 1))).to(xt)
    _, w, _, ws, bias = product_case(3, 1, K, N)
    w8, xg = rows8(w), x.to(DEV)[:, :K]
    neg = T % 2 == 0
    q, scale = rows8(torch.zeros(T, K, dtype=torch.int8)), torch.zeros(T, device=DEV)
    hip.quant_rows(xg, q, scale, lrelu=neg)
    two, one = torch.empty(T, N, device=DEV), torch.empty(T, N, device=DEV)
    hip.gemm_q8(q, scale, w8, ws.to(DEV), two, bias.to(DEV))
    hip.linear_q8(xg, w8, ws.to(DEV), one, rows8(torch.zeros(T, K, dtype=torch.int8)), torch.zeros(T, device=DEV), bias.to(DEV), lrelu=neg)
    assert torch.equal(one, two)
    cq, cs = codes_of(lrelu(x[:, :K].float()) if neg else x[:, :K].float())
    want, tol = product64(cq, cs, w, ws, bias)
    check_product(one, want, tol, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 16, 40, 200])
def test_rows_that_are_not_finite_touch_their_own_row_only(hip, T):
    rng = np.random.default_rng(1)
    K, N = 200, 90
    x = rnd(rng, T, K)
    _, w, _, ws, _ = product_case(3, 1, K, N)
    run = lambda x: (lambda y: (hip.linear_q8(x.to(DEV), rows8(w), ws.to(DEV), y, rows8(torch.zeros(T, K, dtype=torch.int8)),
                                              torch.zeros(T, device=DEV)), y)[1])(torch.empty(T, N, device=DEV))
    clean = run(x)
    x[T // 2, 7] = float("inf")
    x[T - 1, 199] = float("nan")
    got = run(x)
    bad = sorted({T // 2, T - 1})
    rest = [t for t in range(T) if t not in bad]
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[rest], clean[rest])


@pytest.mark.gpu
def test_no_rows(hip):
    _, w, _, ws, _ = product_case(3, 1, 32, 16)
    e8, ef = torch.empty(0, 32, dtype=torch.int8, device=DEV), torch.empty(0, device=DEV)
    y = torch.empty(0, 16, device=DEV)
    hip.quant_rows(torch.empty(0, 32, device=DEV), e8, ef)
    hip.gemm_q8(e8, ef, rows8(w), ws.to(DEV), y)
    hip.linear_q8(torch.empty(0, 32, device=DEV), rows8(w), ws.to(DEV), y, e8, ef)
    hip.up_fold_q8(torch.empty(0, 4, 4, 16 * 32, device=DEV), None, e8, ef)
    hip.up_fold(torch.empty(0, 4, 4, 16 * 32, device=DEV), None, torch.empty(0, 8, 8, 32, device=DEV))


# ---- the fold ------------------------------------------------------------------------------------------------------
FOLDS = [(1, 1, 1, 1), (1, 8, 8, 128), (2, 4, 4, 256), (3, 5, 7, 64), (1, 3, 2, 65), (2, 1, 9, 8), (2, 6, 1, 33), (1, 2, 2, 512), (1, 2, 3, 700),
         (2, 32, 32, 1), (3, 5, 3, 1), (1, 16, 16, 64), (2, 3, 3, 16), (1, 4, 5, 100), (1, 2, 2, 2000), (5, 9, 11, 2), (1, 7, 7, 24)]


def fold64(y, shift):
    """ConvTranspose2d's definition with an identity for its product: every (kh, kw, c) column of y goes to 2 i + k - 1."""
    B, H, W, C16 = y.shape
    C = C16 // 16
    t = y.double().view(B, H, W, 4, 4, C).permute(0, 5, 3, 4, 1, 2).reshape(B, C * 16, H * W)
    fold = lambda z: F.fold(z, (2 * H, 2 * W), kernel_size=4, stride=2, padding=1).permute(0, 2, 3, 1)
    o, mag = fold(t), fold(t.abs())
    if shift is not None:
        o, mag = o + shift.double(), mag + shift.double().abs()
    return o, 4 * U * mag


def fold32(y, shift):
    """The same in fp32 in the kernels' order: rows first, then columns, then the shift."""
    B, H, W, C16 = y.shape
    C = C16 // 16
    t = y.float().view(B, H, W, 4, 4, C)
    out = torch.empty(B, 2 * H, 2 * W, C)
    for oh in range(2 * H):
        for ow in range(2 * W):
            def tap(other_h, other_w):
                i, kh = (oh >> 1, 2 if oh & 1 else 1) if not other_h else ((oh >> 1) + (1 if oh & 1 else -1), 0 if oh & 1 else 3)
                j, kw = (ow >> 1, 2 if ow & 1 else 1) if not other_w else ((ow >> 1) + (1 if ow & 1 else -1), 0 if ow & 1 else 3)
                return t[:, i, j, kh, kw] if 0 <= i < H and 0 <= j < W else torch.zeros(B, C)
            out[:, oh, ow] = (tap(0, 0) + tap(1, 0)) + (tap(0, 1) + tap(1, 1))
    return out if shift is None else out + shift


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H,W,C", FOLDS)
def test_up_fold(hip, B, H, W, C, dtype):
    rng = np.random.default_rng(B + H + W + C)
    y, shift = rnd(rng, B, H, W, 16 * C).to(dtype), rnd(rng, C) if C != 33 else None
    want, tol = fold64(y, shift)
    sg = None if shift is None else shift.to(DEV)
    for act in (0, 1, 2):
        out = torch.full((B * 4 * H * W * C + 9,), 7.0, device=DEV)
        hip.up_fold(y.to(DEV), sg, out[:-9].view(B, 2 * H, 2 * W, C), act)
        got = out[:-9].view(B, 2 * H, 2 * W, C).double().cpu()
        assert bool((out[-9:] == 7).all())
        # sigmoid' <= 1/4 and tanh' <= 1 carry the sum's error on; exp, tanh, the addition and the quotient are within a few u
        w = (want, torch.sigmoid(want), torch.tanh(want))[act]
        assert bool(((got - w).abs() <= tol * (1, 0.25, 1)[act] + (0, 8 * U, 8 * U)[act]).all())
    q, scale = rows8(torch.ones(B * 4 * H * W, C, dtype=torch.int8)), torch.zeros(B * 4 * H * W, device=DEV)
    hip.up_fold_q8(y.to(DEV), sg, q, scale)
    cq, cs = codes_of(lrelu(fold32(y, shift)).view(-1, C))
    assert torch.equal(q.cpu(), cq)
    same(scale.cpu(), cs)
    rest_kept(q)


@pytest.mark.gpu
def test_up_fold_q8_of_odd_values(hip):
    rng = np.random.default_rng(2)
    y = rnd(rng, 1, 4, 4, 16 * 64)
    y[0, 1, 1, 5 * 64 + 3] = float("nan")        # tap (1, 1) of pixel (1, 1): output pixel (2, 2) alone
    y[0, 3, 3, 10 * 64] = float("inf")           # tap (2, 2) of pixel (3, 3): output pixel (7, 7)
    y[0, 0, 0, 5 * 64:6 * 64] = 0                # what is left of output pixel (0, 0): nothing but the shift
    q, scale = rows8(torch.ones(64, 64, dtype=torch.int8)), torch.zeros(64, device=DEV)
    hip.up_fold_q8(y.to(DEV), torch.zeros(64, device=DEV), q, scale)
    cq, cs = codes_of(lrelu(fold32(y, None)).view(-1, 64))
    assert torch.equal(q.cpu(), cq)
    same(scale.cpu(), cs)
    assert torch.isnan(scale).nonzero().view(-1).tolist() == [2 * 8 + 2, 7 * 8 + 7] and bool((q[0] == 0).all())


@pytest.mark.gpu
def test_a_captured_product_replays(hip):
    """linear_q8 and a fold in a graph, replayed on new inputs between eager calls on another stream's buffers."""
    rng = np.random.default_rng(5)
    _, w, _, ws, _ = product_case(3, 1, 96, 16 * 32)
    w8, wsg = rows8(w), ws.to(DEV)

    def buffers():
        return dict(x=torch.zeros(16, 96, device=DEV), y=torch.zeros(16, 512, dtype=torch.bfloat16, device=DEV),
                    q=rows8(torch.zeros(16, 96, dtype=torch.int8)), qs=torch.zeros(16, device=DEV),
                    o=rows8(torch.zeros(64, 32, dtype=torch.int8)), os=torch.zeros(64, device=DEV))

    def go(s):
        hip.linear_q8(s["x"], w8, wsg, s["y"], s["q"], s["qs"], lrelu=True)
        hip.up_fold_q8(s["y"].view(1, 4, 4, 512), None, s["o"], s["os"])
    a, b = buffers(), buffers()
    go(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(a)
    side = torch.cuda.Stream()
    for _ in range(4):
        x, z = rnd(rng, 16, 96), rnd(rng, 16, 96)
        a["x"].copy_(x)
        b["x"].copy_(z)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            go(b)
        torch.cuda.synchronize()
        got = [t.clone() for t in (a["y"], a["o"], a["os"], b["y"], b["o"], b["os"])]
        c, d = buffers(), buffers()
        c["x"].copy_(x)
        d["x"].copy_(z)
        go(c)
        go(d)
        torch.cuda.synchronize()
        for g, want in zip(got, (c["y"], c["o"], c["os"], d["y"], d["o"], d["os"])):
            assert torch.equal(g, want)


@pytest.mark.gpu
def test_refusals(hip):
    from pgan_hip import PganError
    x, q, s = torch.zeros(4, 32, device=DEV), torch.zeros(4, 32, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV)
    w, ws, y = torch.zeros(16, 32, dtype=torch.int8, device=DEV), torch.zeros(16, device=DEV), torch.zeros(4, 16, device=DEV)
    odd = torch.zeros(4 * 33, dtype=torch.int8, device=DEV)
    short = torch.zeros(3 * 32 + 20, dtype=torch.int8, device=DEV).as_strided((4, 20), (32, 1))
    for bad in (lambda: hip.quant_rows(x.cpu(), q, s), lambda: hip.quant_rows(x.double(), q, s), lambda: hip.quant_rows(x.t(), q, s),
                lambda: hip.quant_rows(x, q[:3], s), lambda: hip.quant_rows(x, q, s[:3]), lambda: hip.quant_rows(x, q.float(), s),
                lambda: hip.quant_rows(x, odd[1:129].view(4, 32), s), lambda: hip.quant_rows(x, odd.view(4, 33)[:, :32], s),
                lambda: hip.quant_rows(x[:, :20], short, s), lambda: hip.quant_rows(x[:, :0], q[:, :0], s),
                lambda: hip.quant_rows(x[:1].expand(4, 32), q, s),
                lambda: hip.gemm_q8(q, s, w, ws, y[:3]), lambda: hip.gemm_q8(q, s, w[:15], ws, y), lambda: hip.gemm_q8(q, s, w, ws[:15], y),
                lambda: hip.gemm_q8(q, s, w, ws, y, bias=ws[:15]), lambda: hip.gemm_q8(q[:, :16], s, w, ws, y),
                lambda: hip.gemm_q8(q, s.cpu(), w, ws, y), lambda: hip.gemm_q8(q, s, w, ws, y.double()),
                lambda: hip.gemm_q8(q, s, w, ws, torch.zeros(16, 4, device=DEV).t()),
                lambda: hip.gemm_q8(q, y.view(-1)[:4], w, ws, y),
                lambda: hip.linear_q8(x, w, ws, y, q[:3], s), lambda: hip.linear_q8(x, w, ws, x[:, :16], q, s),
                lambda: hip.linear_q8(x[:3], w, ws, y, q, s),
                lambda: hip.up_fold_q8(y.view(1, 1, 4, 16), None, q, s), lambda: hip.up_fold_q8(y.view(1, 2, 2, 16), None, q, s),
                lambda: hip.up_fold(y.view(1, 2, 2, 16), s, torch.zeros(1, 4, 4, 1, device=DEV)),
                lambda: hip.up_fold(y.view(1, 2, 2, 16), None, torch.zeros(1, 4, 4, 1, device=DEV), 3),
                lambda: hip.up_fold(y.view(1, 2, 2, 16), None, torch.zeros(1, 4, 4, 2, device=DEV)),
                lambda: hip.up_fold(y.view(1, 2, 2, 16), None, y.view(1, 4, 4, 4)[..., :1])):
        with pytest.raises(PganError):
            bad()


def test_entry_point_refusals():
    """Bad arguments come back as -1 before anything is launched (no GPU needed); no rows are no work."""
    import pgan_hip
    lib = pgan_hip._lib._real
    a, b, c, d = 4096, 8192, 12288, 16384

    def quant(x=a, xt=0, ldx=32, q=b, ldq=32, s=c, rows=4, K=32):
        return lib.pgan_quant_rows(x, xt, ldx, q, ldq, s, rows, K, 0, None)

    def gemm(q=a, ldq=32, s=b, w=c, ldw=32, ws=d, y=a, yt=0, ldy=16, T=4, N=16, K=32):
        return lib.pgan_gemm_q8(q, ldq, s, w, ldw, ws, None, y, yt, ldy, T, N, K, None)

    def linear(x=a, xt=0, ldx=32, q=b, ldq=32, s=c, w=d, ldw=32, ws=a, y=b, yt=0, ldy=16, T=4, N=16, K=32):
        return lib.pgan_linear_q8(x, xt, ldx, q, ldq, s, w, ldw, ws, None, y, yt, ldy, T, N, K, 0, None)

    def fold8(y=a, yt=0, q=b, ldq=16, s=c, B=1, H=4, W=4, C=16):
        return lib.pgan_up_fold_q8(y, yt, None, q, ldq, s, B, H, W, C, None)

    def fold(y=a, yt=0, o=b, B=1, H=4, W=4, C=16, act=0):
        return lib.pgan_up_fold(y, yt, None, o, B, H, W, C, act, None)
    for fn, bads in ((quant, (dict(x=None), dict(xt=3), dict(xt=-1), dict(ldx=31), dict(q=None), dict(ldq=31), dict(s=None), dict(rows=-1),
                              dict(K=0), dict(x=4098), dict(rows=1 << 40))),
                     (gemm, (dict(q=None), dict(q=a + 8), dict(ldq=40), dict(ldq=16), dict(w=c + 1), dict(ldw=33), dict(ws=None), dict(y=None),
                             dict(yt=3), dict(ldy=15), dict(T=-1), dict(N=0), dict(K=0), dict(K=131073), dict(y=a + 2), dict(T=1 << 42))),
                     (linear, (dict(x=None), dict(xt=5), dict(ldx=8), dict(q=b + 4), dict(ldq=24), dict(s=None), dict(w=None), dict(ldw=31),
                               dict(ldy=15), dict(T=-1), dict(N=0), dict(K=0), dict(K=131073), dict(yt=-1), dict(x=a + 2), dict(T=1 << 42))),
                     (fold8, (dict(y=None), dict(yt=3), dict(q=None), dict(ldq=15), dict(s=None), dict(B=-1), dict(H=0), dict(W=0), dict(C=0),
                              dict(H=40000), dict(y=a + 1), dict(B=1 << 30))),
                     (fold, (dict(y=None), dict(yt=-1), dict(o=None), dict(o=b + 2), dict(B=-1), dict(H=0), dict(W=40000), dict(C=0), dict(act=3),
                             dict(act=-1), dict(B=1 << 30)))):
        for bad in bads:
            assert fn(**bad) == -1, (fn.__name__, bad)
    assert quant(rows=0) == gemm(T=0) == linear(T=0) == fold8(B=0) == fold(B=0) == 0


def test_entry_point_refuses_what_a_launch_cannot_hold():
    """Rows whose places a 32-bit loop would run past, and more channels than a launch has threads for (no GPU needed)."""
    import pgan_hip
    lib = pgan_hip._lib._real
    a, b, c, d, far = 1 << 12, 1 << 40, 1 << 44, 1 << 45, 1 << 46
    big = (1 << 30) + 1
    assert lib.pgan_quant_rows(a, 1, big, b, big, c, 1, big, 0, None) == -1
    assert lib.pgan_up_fold_q8(a, 1, None, b, big, c, 1, 1, 1, big, None) == -1
    assert lib.pgan_up_fold(a, 1, None, b, 1, 1, 1, big, 0, None) == -1
    n = 1 << 29
    assert lib.pgan_gemm_q8(a, 16, b, c, 16, d, None, far, 1, n, 1, n, 16, None) == -1
    assert lib.pgan_linear_q8(a, 1, 16, b, 16, c, d, 16, 1 << 47, None, far, 1, n, 1, n, 16, 0, None) == -1


@pytest.mark.gpu
def test_offsets_past_31_bits(hip):
    """Rows, codes, results and taps whose last places lie past 2^31 elements; the first and last rows against the definition."""
    rng = np.random.default_rng(2)
    T, K, N = 270000, 8192, 40
    x = torch.full((T, K), 0.5, dtype=torch.bfloat16, device=DEV)
    q, s = torch.zeros(T, K, dtype=torch.int8, device=DEV), torch.zeros(T, device=DEV)
    ends = torch.cat([torch.arange(3), torch.arange(T - 3, T)])
    x[ends.to(DEV)] = rnd(rng, 6, K).to(torch.bfloat16).to(DEV)
    hip.quant_rows(x, q, s)
    want, ws = codes_of(x[ends.to(DEV)].float().cpu())
    assert torch.equal(q[ends.to(DEV)].cpu(), want)
    same(s[ends.to(DEV)].cpu(), ws)
    _, w, _, wscale, bias = product_case(4, 1, K, N)
    y = torch.zeros(T, N, device=DEV)
    hip.gemm_q8(q, s, w.to(DEV), wscale.to(DEV), y, bias.to(DEV))
    out, tol = product64(want, ws, w, wscale, bias)
    check_product(y[ends.to(DEV)], out, tol, torch.float32)
    del x, q, y
    T, K, N = 70000, 64, 32768
    q, w, qs, wscale, bias = product_case(5, T, K, N)
    y = torch.zeros(T, N, dtype=torch.bfloat16, device=DEV)
    hip.gemm_q8(q.to(DEV), qs.to(DEV), w.to(DEV), wscale.to(DEV), y, bias.to(DEV))
    ends = torch.cat([torch.arange(3), torch.arange(T - 3, T)])
    out, tol = product64(q[ends], qs[ends], w, wscale, bias)
    check_product(y[ends.to(DEV)], out, tol, torch.bfloat16)
    del y
    B, H, W, C = 33000, 16, 16, 16
    y = torch.full((B, H, W, 16 * C), 0.25, dtype=torch.bfloat16, device=DEV)
    part = rnd(rng, 1, H, W, 16 * C).to(torch.bfloat16)
    y[-1] = part[0].to(DEV)
    q, s = torch.zeros(4 * B * H * W, C, dtype=torch.int8, device=DEV), torch.zeros(4 * B * H * W, device=DEV)
    hip.up_fold_q8(y, None, q, s)
    want, ws = codes_of(lrelu(fold32(part, None)).view(-1, C))
    assert torch.equal(q[-4 * H * W:].cpu(), want)
    same(s[-4 * H * W:].cpu(), ws)
    one = torch.full((2100000, 8, 8, 16), 0.25, dtype=torch.bfloat16, device=DEV)
    part = rnd(rng, 1, 8, 8, 16).to(torch.bfloat16)
    one[-1] = part[0].to(DEV)
    out = torch.zeros(2100000, 16, 16, 1, device=DEV)
    hip.up_fold(one, None, out)
    assert torch.equal(out[-1:].cpu(), fold32(part, None))
    del one, out, y, q, s
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [1025, 1032, 2047, 2056, 4097, 4104, 8190, 8192, 8200])
def test_quant_rows_of_more_than_a_wave(hip, K, dtype):
    """Rows of a block, on borders of 16 bytes and of one element, an infinity and a NaN in their last elements."""
    rng = np.random.default_rng(K)
    x = rnd(rng, 9, K) * torch.exp(2 * rnd(rng, 9, 1))
    x[3, K - 1], x[5, K - 2] = float("inf"), float("nan")
    x[7, K - 1] = 100.0
    x = x.to(dtype)
    for gap in (0, 1, 16 - K % 8):
        for neg in (False, True):
            view = torch.full((9, K + gap), float("nan"), dtype=dtype, device=DEV)[:, :K]
            view.copy_(x.to(DEV))
            want, ws = codes_of(lrelu(x.float()) if neg else x.float())
            q, s = rows8(torch.zeros(9, K, dtype=torch.int8)), torch.zeros(9, device=DEV)
            hip.quant_rows(view, q, s, lrelu=neg)
            assert torch.equal(q.cpu(), want)
            same(s.cpu(), ws)
            rest_kept(q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_every_operand_on_borders_of_one_element(hip, dtype):
    """Rows of x and y that start anywhere in memory, with odd strides; what lies between and around y's rows stays."""
    rng = np.random.default_rng(12)
    for T, K, N in ((1, 5, 3), (7, 200, 90), (30, 700, 130), (21, 300, 1000), (70, 1001, 257), (300, 129, 640), (5000, 65, 33), (6500, 70, 1301)):
        x = (rnd(rng, T, K) * torch.exp(rnd(rng, T, 1))).to(dtype)
        _, w, _, ws, bias = product_case(T, 1, K, N)
        ldx, ldy = K + 1 + K % 2 * 2, N + 3 - N % 2
        assert ldy % 2 == 1 or N % 2 == 0
        xb = torch.full((T * ldx + 1,), float("nan"), dtype=dtype, device=DEV)
        xv = xb[1:].view(T, ldx)[:, :K]
        xv.copy_(x.to(DEV))
        yb = torch.full((T * ldy + 1,), 7.0, dtype=dtype, device=DEV)
        yv = yb[1:].view(T, ldy)[:, :N]
        q, s = rows8(torch.zeros(T, K, dtype=torch.int8)), torch.zeros(T, device=DEV)
        hip.linear_q8(xv, rows8(w), ws.to(DEV), yv, q, s, bias.to(DEV), lrelu=True)
        want, tol = product64(*codes_of(lrelu(x.float())), w, ws, bias)
        check_product(yv, want, tol, dtype)
        assert float(yb[0]) == 7 and bool((yb[1:].view(T, ldy)[:, N:] == 7).all())
        q2, s2 = rows8(torch.zeros(T, K, dtype=torch.int8)), torch.zeros(T, device=DEV)
        hip.quant_rows(xv, q2, s2, lrelu=True)
        qw, sw = codes_of(lrelu(x.float()))
        assert torch.equal(q2.cpu(), qw) and torch.equal(s2.cpu(), sw)
        rest_kept(q2)
    for B, H, W, C in ((2, 3, 5, 1), (1, 4, 3, 5), (2, 2, 2, 13), (1, 3, 2, 64), (1, 2, 2, 333), (1, 1, 2, 700)):
        y, shift = rnd(rng, B, H, W, 16 * C).to(dtype), rnd(rng, C)
        yb = torch.full((y.numel() + 2,), float("nan"), dtype=dtype, device=DEV)
        yv = yb[1:-1].view(y.shape)
        yv.copy_(y.to(DEV))
        ob = torch.full((4 * B * H * W * C + 2,), 7.0, device=DEV)
        ov = ob[1:-1].view(B, 2 * H, 2 * W, C)
        hip.up_fold(yv, shift.to(DEV), ov)
        assert torch.equal(ov.cpu(), fold32(y, shift)) and float(ob[0]) == 7 and float(ob[-1]) == 7
        q, s = rows8(torch.zeros(4 * B * H * W, C, dtype=torch.int8)), torch.zeros(4 * B * H * W, device=DEV)
        hip.up_fold_q8(yv, shift.to(DEV), q, s)
        qw, sw = codes_of(lrelu(fold32(y, shift)).view(-1, C))
        assert torch.equal(q.cpu(), qw) and torch.equal(s.cpu(), sw)
        rest_kept(q)


@pytest.mark.gpu
def test_rows8_buffers(hip):
    """What pgan_hip.rows8 gives: zeros, rows that a product takes, from 128 columns on one to a run of 128-byte lines."""
    from pgan_hip import rows8 as buffer
    for T, K in ((3, 1), (2, 16), (5, 127), (1, 128), (4, 129), (3, 1000), (0, 40)):
        b = buffer(T, K, DEV)
        assert b.shape == (T, K) and b.dtype == torch.int8 and b.stride(0) % (128 if K >= 128 else 16) == 0 and not bool(b.any())
        s, w, ws, y = torch.ones(max(T, 1), device=DEV), buffer(6, K, DEV), torch.ones(6, device=DEV), torch.ones(T, 6, device=DEV)
        w.fill_(1)
        b.fill_(2)
        hip.gemm_q8(b, s, w, ws, y)
        assert torch.equal(y, torch.full_like(y, 2.0 * K))


def test_one_launch_codes_every_token():
    """Where linear_q8 is one launch, each block's waves make the codes of at least as many rows as there are tokens (no GPU
    needed: the rule that the launch is made by, over every K that a product takes and every T that it can hold)."""
    import pgan_hip
    rows = pgan_hip._lib.pgan_linear_q8_rows
    one = set()
    for K in list(range(1, 4200)) + [k for b in range(4096, 131072, 512) for k in (b + 511, b + 512, b + 513) if k <= 131072]:
        for T in range(1, 41):
            n = rows(T, K)
            assert n == 0 or n >= T, (T, K, n)
            if n:
                one.add((T, K))
    # both sides of each border are there
    for T, K in ((1, 1), (32, 256), (16, 257), (16, 512), (8, 513), (8, 1023), (8, 1024), (8, 1025), (8, 2048)):
        assert (T, K) in one, (T, K)
    for T, K in ((33, 16), (17, 257), (17, 512), (9, 513), (9, 1023), (17, 1024), (9, 1025), (9, 2048), (1, 2049), (1, 131072)):
        assert (T, K) not in one, (T, K)
    assert rows(0, 16) == rows(-1, 16) == rows(1, 0) == rows(1, -5) == rows(1 << 40, 16) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("K", [8, 16, 256, 257, 512, 513, 1000, 1023, 1024, 1025, 1536, 2048, 2049])
@pytest.mark.parametrize("xt,yt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_linear_q8_at_the_borders_of_one_launch(hip, K, xt, yt):
    """Every number of tokens next to a border of the rule, bit for bit what rows to codes and the product give one after the
    other, and that of the definition; what a block's LDS held before is other rows' codes and scales."""
    rng = np.random.default_rng(K)
    N = 70
    _, w, _, ws, bias = product_case(K, 1, K, N)
    w8, wsg, bg = rows8(w), ws.to(DEV), bias.to(DEV)
    for T in (1, 4, 5, 7, 8, 9, 12, 15, 16, 17, 31, 32):
        x = (rnd(rng, T, K) * torch.exp(2 * rnd(rng, T, 1))).to(xt)
        xg, neg = x.to(DEV), T % 2 == 1
        q, s = rows8(torch.zeros(T, K, dtype=torch.int8)), torch.zeros(T, device=DEV)
        two, one = (torch.full((T + 1, N), 7.0, dtype=yt, device=DEV) for _ in range(2))
        hip.quant_rows(xg, q, s, lrelu=neg)
        hip.gemm_q8(q, s, w8, wsg, two[:T], bg)
        hip.linear_q8(torch.full((32, K), 1e4, dtype=xt, device=DEV), w8, wsg, torch.empty(32, N, dtype=yt, device=DEV),
                      rows8(torch.zeros(32, K, dtype=torch.int8)), torch.zeros(32, device=DEV))
        hip.linear_q8(xg, w8, wsg, one[:T], rows8(torch.zeros(T, K, dtype=torch.int8)), torch.zeros(T, device=DEV), bg, lrelu=neg)
        assert torch.equal(one, two), (T, K)
        want, tol = product64(*codes_of(lrelu(x.float()) if neg else x.float()), w, ws, bias)
        check_product(one[:T], want, tol, yt)


def test_a_launch_of_too_many_threads_is_refused():
    """Every tiling's launch stays below 2^32 threads (no GPU needed: refused before anything is launched)."""
    import pgan_hip
    lib = pgan_hip._lib._real
    q, s, w, ws, y, x = 1 << 12, 1 << 40, 1 << 41, 1 << 42, 1 << 46, 1 << 44
    for T, N in ((1 << 30, 129), (715827968, 257), ((1 << 31) - 256, 200)):
        assert lib.pgan_gemm_q8(q, 16, s, w, 16, ws, None, y, 1, N, T, N, 16, None) == -1, (T, N)
        assert lib.pgan_linear_q8(x, 1, 16, q, 16, s, w, 16, ws, None, y, 1, N, T, N, 16, 0, None) == -1, (T, N)
