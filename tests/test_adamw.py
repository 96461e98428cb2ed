"""AdamW over many tensors (pgan_adamw_multi): states in 32 and in 8 bits against the formulas in 64 bits, its refusals, its
replay from a graph and from a launch tape.

Tolerances: u = 2^-24 is the largest relative error of one fp32 rounding.  m = b1 m + c1 g takes a rounding of each constant,
of each product and of the sum: at most 3 u (|b1 m| + |c1 g|) to first order; v likewise with one product more, 4 u of a sum
of positive terms; 4 and 5 are used.  p keep - upd: keep's rounding, the product's and the difference's on p (3 u |p|, plus
u |upd|), and on upd = size m / (sqrt(v) inv + eps) the error of m, half of v's (2.5 u), and one rounding each of size, its
product, the root, inv, its product, eps, the sum and the quotient: 4 u of m's terms and 11 u of upd; 16 is used.  A result
in fewer bits adds half a step of its type."""
import ctypes
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
M32 = 0xFFFFFFFF
BLOCK = 256
B1, B2, EPS = 0.5, 0.999, 1e-8
DEV = "cuda:0"


@pytest.fixture(scope="module")
def hip():
    from pgan_hip import HipOps
    return HipOps(torch.device(DEV), ws_floats=4, max_samples=1)


# ---- the formulas --------------------------------------------------------------------------------------------------
def _mix(x):
    x = ((x ^ (x >> 16)) * 0x6A09E667) & M32
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def random_bits(n, seed, step, index):
    key = _mix((seed + step * 0xA54FF53B + index * 0x3C6EF373) & M32)
    h = _mix(torch.full((n,), key, dtype=torch.int64) ^ (torch.arange(n) & M32))
    return h & 0xFFFF, h >> 16


def blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def exponent(x):
    return (x.view(torch.int32) >> 23) - 127


def encode(y, u16):
    small = y < 2.0 ** -6
    bits = torch.where(small, y + 2.0 ** -6, y).view(torch.int32).to(torch.int64)
    return ((bits + (u16 << 4) + 8) >> 20) - 960 - 8 * small


def hold8(m, v, seed, step, index):
    """Codes and scales of the new states (fp32, this format's definition)."""
    mb, vb = blocks(m), blocks(v)
    um, ur = (blocks(u) for u in random_bits(m.numel(), seed, step, index))
    fine_m, fine_v = torch.isfinite(mb), torch.isfinite(vb)
    em = exponent(torch.where(fine_m, mb.abs(), 0.0).amax(1)).clamp_min(-100) - 7
    er = (exponent(torch.where(fine_v, vb, 0.0).amax(1)).clamp_min(-126) >> 1) - 7
    one = torch.ones(1)
    ms, rs = torch.ldexp(one, em), torch.ldexp(one, er)
    cm = torch.where(fine_m, encode(torch.where(fine_m, mb.abs(), 0.0) * torch.ldexp(one, -em)[:, None], um), 0x7F)
    cm = cm + 128 * (mb.view(torch.int32) < 0)
    cr = torch.maximum(encode(torch.where(fine_v, vb, 0.0).sqrt() * torch.ldexp(one, -er)[:, None], ur), (vb > 0).to(torch.int64))
    cr = torch.where(fine_v, cr, 0x7F)
    n = m.numel()
    return cm.to(torch.uint8).view(-1)[:n], cr.to(torch.uint8).view(-1)[:n], ms, rs


def values8(code, scale):
    """Values of codes (a uint8 tensor) with their blocks' scales, fp32."""
    v = blocks(code).view(torch.float8_e4m3fn).float() * scale[:, None]
    return v.view(-1)[:code.numel()]


def states32(m, v, g, b1=B1, b2=B2):
    """m and v of the definition, rounded one by one in fp32."""
    return m * b1 + g * (1 - b1), v * b2 + (g * g) * (1 - b2)


def step64(p, g, m, v, t, lr, wd, gs=1.0):
    p, g, m, v = p.double(), g.double() * gs, m.double(), v.double()
    mn, vn = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    upd = lr / (1 - B1 ** t) * mn / (vn.sqrt() / math.sqrt(1 - B2 ** t) + EPS)
    size = lr / (1 - B1 ** t) / (vn.sqrt() / math.sqrt(1 - B2 ** t) + EPS)
    terms = (B1 * m).abs() + ((1 - B1) * g).abs()
    return p * (1 - lr * wd) - upd, mn, vn, terms, size * 4 * U * terms + 16 * U * upd.abs() + 4 * U * p.abs()


def within(name, got, want, tol):
    got, want = got.double().cpu(), want.cpu()
    bad = ~((got - want).abs() <= tol.cpu() + 1e-45)
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} outside, worst {float((got - want).abs().max())}"


def half_step(x, dtype):
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[dtype]
    return torch.finfo(dtype).eps / 2 * x.abs() * (dtype != torch.float32) + least


SIZES = [1, 3, 64, 255, 256, 257, 1000, 2048, 2049, 5003]


def make(seed, sizes, pt=torch.float32, gt=torch.float32, bits=32, offset=0):
    """Tensors on the CPU; views `offset` elements into their storage, which ends in guard values."""
    rng = np.random.default_rng(seed)
    rnd = lambda n, s: torch.from_numpy((rng.standard_normal(n) * s).astype(np.float32))
    out = dict(p=[], g=[], m=[], v=[], ms=[], rs=[])
    for n in sizes:
        out["p"].append(rnd(n, 0.05).to(pt))
        out["g"].append((rnd(n, 1e-3) * torch.exp(rnd(n, 2.0))).to(gt))
        m, v = rnd(n, 1e-3), rnd(n, 1e-3).square()
        if bits == 8:
            m, v, ms, rs = hold8(m, v, 3, 1, 0)
            out["ms"].append(ms)
            out["rs"].append(rs)
        out["m"].append(m)
        out["v"].append(v)
    return out


GUARD = 17


def on_gpu(t, offset=0):
    """A view of a longer buffer: `offset` elements before it, GUARD after."""
    raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    buf = torch.full((raw.numel() + offset + GUARD,), 85, dtype=raw.dtype)
    buf[offset:offset + raw.numel()] = raw
    return buf.to(DEV)[offset:offset + raw.numel()]


def guards_kept(view, offset):
    base = view._base if view._base is not None else view
    base = base.view(torch.uint8) if base.dtype == torch.float8_e4m3fn else base
    n = view.numel()
    flat = base.reshape(-1).cpu()
    assert bool((flat[:offset].double() == 85).all()) and bool((flat[offset + n:].double() == 85).all())


def run(hip, d, bits, t, lr=1e-3, wd=0.01, seed=7, offset=0, gs=1.0, step_dev=None):
    gpu = {k: [on_gpu(x, offset if k in ("p", "g", "m", "v") else 0) for x in d[k]] for k in d}
    m, v = gpu["m"], gpu["v"]
    if bits == 8:
        m, v = [x.view(torch.float8_e4m3fn) for x in m], [x.view(torch.float8_e4m3fn) for x in v]
    hip.adamw(gpu["p"], gpu["g"], m, v, t, lr, B1, B2, EPS, wd, scales=(gpu["ms"], gpu["rs"]) if bits == 8 else None, seed=seed,
              grad_scale=gs, step_dev=step_dev)
    torch.cuda.synchronize()
    for k in ("p", "g", "m", "v"):
        for x in gpu[k]:
            guards_kept(x, offset)
    return gpu


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("pt,gt", [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float32"),
                                   ("bfloat16", "float16"), ("float16", "float16")])
def test_states_in_32_bits(hip, pt, gt, offset):
    pt, gt = getattr(torch, pt), getattr(torch, gt)
    d = make(1, SIZES, pt, gt)
    got = run(hip, d, 32, 5, offset=offset, gs=0.5)
    for i in range(len(SIZES)):
        p, m, v, terms, tol = step64(d["p"][i], d["g"][i], d["m"][i], d["v"][i], 5, 1e-3, 0.01, 0.5)
        within("m", got["m"][i], m, 4 * U * terms)
        within("v", got["v"][i], v, 5 * U * v)
        within("p", got["p"][i], p, tol + half_step(p.abs() + tol, pt))


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("pt,gt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("float32", "float16")])
def test_states_in_8_bits(hip, pt, gt, offset):
    """The codes are those of the format's definition, bit for bit, and each is one of the two neighbours of the 64-bit
    value; the parameters are those of the 64-bit formulas."""
    pt, gt = getattr(torch, pt), getattr(torch, gt)
    d = make(2, SIZES, pt, gt, bits=8)
    got = run(hip, d, 8, 5, offset=offset, seed=99)
    for i, n in enumerate(SIZES):
        m, r = values8(d["m"][i], d["ms"][i]), values8(d["v"][i], d["rs"][i])
        p, m64, v64, terms, tol = step64(d["p"][i], d["g"][i], m, r * r, 5, 1e-3, 0.01)
        within("p", got["p"][i], p, tol + half_step(p.abs() + tol, pt))
        cm, cr, ms, rs = hold8(*states32(m, r * r, d["g"][i].float()), 99, 5, i)
        assert torch.equal(got["ms"][i].cpu(), ms) and torch.equal(got["rs"][i].cpu(), rs)
        assert torch.equal(got["m"][i].cpu(), cm) and torch.equal(got["v"][i].cpu(), cr)
        for code, scale, want in ((cm, ms, m64), (cr, rs, v64.sqrt())):
            held, s = values8(code, scale).double(), scale.double().repeat_interleave(BLOCK)[:n]
            step = torch.maximum(want.abs() / 8, s * 2.0 ** -9) * (1 + 2.0 ** -16)      # three bits of mantissa
            within("code", held, want, step)


@pytest.mark.gpu
def test_more_tensors_than_a_launch_holds_and_empty_ones(hip):
    sizes = [int(x) for x in np.random.default_rng(3).integers(0, 3000, 97)]
    sizes[5] = sizes[50] = 0
    lrs, wds = [1e-3 * (i + 1) for i in range(97)], [0.01 * (i % 3) for i in range(97)]
    d = make(4, sizes)
    got = run(hip, d, 32, 3, lr=lrs, wd=wds)
    for i in range(97):
        p, m, v, terms, tol = step64(d["p"][i], d["g"][i], d["m"][i], d["v"][i], 3, lrs[i], wds[i])
        within("p", got["p"][i], p, tol)
        within("v", got["v"][i], v, 5 * U * v)


@pytest.mark.gpu
def test_mixed_types_in_one_list(hip):
    kinds = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)] * 2
    parts = [make(10 + i, [700 + i], *k) for i, k in enumerate(kinds)]
    d = {key: [x for q in parts for x in q[key]] for key in parts[0]}
    got = run(hip, d, 32, 2)
    for i, (pt, _) in enumerate(kinds):
        p, _, _, _, tol = step64(d["p"][i], d["g"][i], d["m"][i], d["v"][i], 2, 1e-3, 0.01)
        within("p", got["p"][i], p, tol + half_step(p.abs() + tol, pt))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite_touch_their_own_elements_only(hip, bits):
    d = make(6, [600], bits=bits)
    clean = run(hip, d, bits, 4)
    at = [0, 100, 256, 599]
    for k, x in zip(at, (math.nan, math.inf, -math.inf, math.nan)):
        d["g"][0][k] = x
    got = run(hip, d, bits, 4)
    rest = torch.ones(600, dtype=torch.bool)
    rest[at] = False
    assert bool(torch.isnan(got["p"][0].cpu()[at]).all())
    assert torch.equal(got["p"][0].cpu()[rest], clean["p"][0].cpu()[rest])
    if bits == 8:
        assert bool(((got["m"][0].cpu()[at] & 0x7F) == 0x7F).all()) and bool((got["v"][0].cpu()[at] == 0x7F).all())
        m, r = values8(d["m"][0], d["ms"][0]), values8(d["v"][0], d["rs"][0])
        cm, cr, ms, rs = hold8(*states32(m, r * r, d["g"][0]), 7, 4, 0)
        assert torch.equal(got["ms"][0].cpu(), ms) and torch.equal(got["rs"][0].cpu(), rs)
        assert torch.equal(got["m"][0].cpu()[rest], cm[rest]) and torch.equal(got["v"][0].cpu()[rest], cr[rest])
    else:
        assert torch.equal(got["m"][0].cpu()[rest], clean["m"][0].cpu()[rest])


@pytest.mark.gpu
def test_a_fresh_8_bit_state_is_zeros_and_small_roots_stay_above_zero(hip):
    n = 512
    g = torch.zeros(n)
    g[0], g[1], g[2] = 1.0, 1e-12, 1e-3          # one block: 1e-12 is far below the block's smallest code
    d = dict(p=[torch.ones(n)], g=[g], m=[torch.zeros(n, dtype=torch.uint8)], v=[torch.zeros(n, dtype=torch.uint8)],
             ms=[torch.zeros(2)], rs=[torch.zeros(2)])
    got = run(hip, d, 8, 1)
    p, _, _, _, tol = step64(d["p"][0], g, torch.zeros(n), torch.zeros(n), 1, 1e-3, 0.01)
    within("p", got["p"][0], p, tol)
    codes = got["v"][0].cpu()
    assert int(codes[1]) >= 1 and bool((codes[3:] == 0).all())
    assert torch.isfinite(got["ms"][0]).all() and torch.isfinite(got["rs"][0]).all()


@pytest.mark.gpu
def test_8_bit_rounding_is_unbiased(hip):
    """n elements with the same m between two codes: the mean of what is held misses m by the spread of n independent
    roundings, at most half a step each (variance <= step^2 / 4): five standard deviations of the mean.  The random bits
    (16 of them) add at most 2^-17 of a step."""
    n = 1 << 16
    for value in (0.3, 0.0123, 1.0 / 3):
        d = dict(p=[torch.zeros(n)], g=[torch.full((n,), value)], m=[torch.zeros(n, dtype=torch.uint8)],
                 v=[torch.zeros(n, dtype=torch.uint8)], ms=[torch.zeros(n // 256)], rs=[torch.zeros(n // 256)])
        got = run(hip, d, 8, 1, seed=31)
        for code, scale, want in ((got["m"][0], got["ms"][0], value * (1 - B1)), (got["v"][0], got["rs"][0], value * math.sqrt(1 - B2))):
            held = values8(code.cpu(), scale.cpu()).double()
            step = want / 8
            assert len(set(held.tolist())) == 2
            assert abs(float(held.mean()) - want) <= 5 * step / 2 / math.sqrt(n) + step * 2.0 ** -17 + want * 4 * U


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_device_counter_in_a_replayed_graph_and_on_a_tape(hip, bits):
    """Five steps counted on the device -- eager, from a graph and from a launch tape -- against five numbered ones."""
    import pgan_tape
    sizes = [300, 1, 5000]
    d = make(8, sizes, bits=bits)
    grads = [make(20 + k, sizes)["g"] for k in range(5)]
    view = (lambda ts: [x.view(torch.float8_e4m3fn) for x in ts]) if bits == 8 else (lambda ts: ts)

    def fresh():
        s = {k: [x.clone().to(DEV) for x in d[k]] for k in d}
        s["g"] = [torch.zeros(n, device=DEV) for n in sizes]
        s["plan"] = hip.adamw_plan(s["p"], view(s["m"]), view(s["v"]), scales=(s["ms"], s["rs"]) if bits == 8 else None)
        return s

    def result(s):
        torch.cuda.synchronize()
        return [x.cpu() for k in ("p", "m", "v", "ms", "rs") for x in s[k]]

    def load(s, k):
        for x, y in zip(s["g"], grads[k]):
            x.copy_(y)
    want = fresh()
    for k in range(5):
        load(want, k)
        want["plan"].step(want["g"], k + 1, 1e-3, B1, B2, EPS, 0.01, seed=5)
    want = result(want)

    def close(got):
        for a, b in zip(got, want):      # the corrections pass through fp32: size and inv differ by a rounding each
            if a.dtype == torch.uint8:
                assert torch.equal(a, b)
            else:
                assert torch.allclose(a, b, rtol=0, atol=5 * 1e-3 * 8 * U + 4 * U) or torch.equal(a, b)

    for how in ("eager", "graph", "tape"):
        s = fresh()
        counter = torch.zeros(4, dtype=torch.int32, device=DEV)
        one = lambda: s["plan"].step(s["g"], 0, 1e-3, B1, B2, EPS, 0.01, seed=5, step_dev=counter)
        if how == "graph":
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                one()
            call = g.replay
        elif how == "tape":
            load(s, 0)
            pgan_tape.tape = []
            try:
                one()                    # recorded while it runs: the first step
            finally:
                entries, pgan_tape.tape = pgan_tape.tape, None
            tape = pgan_tape.compile(entries)
            assert tape.native_calls == 1
            call = tape.replay
        else:
            call = one
        for k in range(1 if how == "tape" else 0, 5):
            load(s, k)
            call()
            torch.cuda.synchronize()
        assert int(counter[0]) == 5
        close(result(s))


@pytest.mark.gpu
def test_plan_refusals_on_the_gpu(hip):
    from pgan_hip import PganError
    p = [torch.zeros(300, device=DEV)]
    m, v = [torch.zeros(300, device=DEV)], [torch.zeros(300, device=DEV)]
    f8 = [torch.zeros(300, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    s = torch.zeros(2, device=DEV)
    bad = [(p, m[:0], v, None), ([p[0].double()], m, v, None), ([torch.zeros(300)], m, v, None), ([torch.zeros(600, device=DEV)[::2]], m, v, None),
           (p, [m[0][:299]], v, None), (p, [m[0].half()], v, None), (p, f8[:1], f8[1:], None), (p, m, v, ([s], [s])),
           (p, f8[:1], f8[1:], ([s], [s[:1]])), (p, f8[:1], f8[1:], ([s.half()], [s])), (p, f8[:1], f8[1:], [[s]])]
    for args in bad:
        with pytest.raises(PganError):
            hip.adamw_plan(*args)
    plan = hip.adamw_plan(p, m, v)
    g = torch.zeros(300, device=DEV)
    for grads, step, more in (([], 1, {}), ([g[:10]], 1, {}), ([torch.zeros(300)], 1, {}), ([g.double()], 1, {}), ([g], 0, {}),
                              ([torch.zeros(600, device=DEV)[::2]], 1, {}), ([g], 1, dict(lr=[1.0, 2.0])),
                              ([g], 0, dict(step_dev=torch.zeros(1, dtype=torch.int32, device=DEV)))):
        with pytest.raises(PganError):
            plan.step(grads, step, more.pop("lr", 1e-3), B1, B2, EPS, 0.0, **more)
    with pytest.raises(PganError):
        plan.step([g], 1, 1e-3, 1.0, B2, EPS)
    twice = hip.adamw_plan(p + p, m + [torch.zeros(300, device=DEV)], v + [torch.zeros(300, device=DEV)])
    with pytest.raises(PganError):       # one tensor twice: two blocks would write it
        twice.step([g, g], 1, 1e-3, B1, B2, EPS)
    both = hip.adamw_plan(p, m, m)       # one state for both
    with pytest.raises(PganError):
        both.step([g], 1, 1e-3, B1, B2, EPS)


def test_entry_point_refusals():
    """Bad arguments come back as -1 before anything is launched (no GPU needed)."""
    import pgan_hip
    fn = pgan_hip._lib._real.pgan_adamw_multi
    P, LL, I, D = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_double
    one = lambda t, x: (t * 1)(x)

    def call(**k):
        a = dict(p=one(P, 4096), g=one(P, 1 << 16), m=one(P, 1 << 20), v=one(P, 1 << 21), ms=None, rs=None, n=one(LL, 100), t=one(I, 0),
                 lr=one(D, 1e-3), wd=one(D, 0.0), k=1, bits=32, b1=0.5, b2=0.999, eps=1e-8, step=1)
        a.update(k)
        return fn(a["p"], a["g"], a["m"], a["v"], a["ms"], a["rs"], a["n"], a["t"], a["lr"], a["wd"], a["k"], a["bits"], a["b1"],
                  a["b2"], a["eps"], 1.0, 0, None, a["step"], None)
    for bad in (dict(k=-1), dict(bits=16), dict(b1=1.0), dict(b1=-0.1), dict(b2=math.nan), dict(eps=-1.0), dict(eps=math.nan), dict(step=0),
                dict(p=None), dict(lr=None), dict(n=one(LL, -1)), dict(n=one(LL, 1 << 40)), dict(t=one(I, 9)), dict(t=one(I, -1)),
                dict(p=one(P, 4098)), dict(m=one(P, (1 << 20) + 2)), dict(bits=8), dict(p=one(P, None)), dict(m=one(P, 4096 + 396)),
                dict(v=one(P, 1 << 20)), dict(bits=8, ms=one(P, 1 << 22), rs=one(P, None)),
                dict(bits=8, ms=one(P, 1 << 22), rs=one(P, 1 << 22))):
        assert call(**bad) == -1, bad
    if not torch.cuda.is_available():
        return
    assert call(k=0) == 0


def test_a_gradient_may_not_share_memory_with_what_is_written():
    """(No GPU needed: refused before anything is launched.)  Nor may the device's step counter."""
    import pgan_hip
    fn = pgan_hip._lib._real.pgan_adamw_multi
    P, LL, I, D = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_double
    two = lambda t, x, y: (t * 2)(x, y)
    p, m, v, s, r = two(P, 4096, 1 << 16), two(P, 1 << 20, 1 << 21), two(P, 1 << 22, 1 << 23), two(P, 1 << 24, 1 << 25), two(P, 1 << 26, 1 << 27)

    def call(g0, g1, bits=32, counter=None):
        return fn(p, two(P, g0, g1), m, v, s, r, two(LL, 100, 300), two(I, 0, 0), two(D, 1e-3, 1e-3), two(D, 0.0, 0.0), 2, bits, 0.5, 0.999,
                  1e-8, 1.0, 0, counter, 1, None)
    free = 1 << 28
    for bits in (32, 8):
        for g0, g1 in ((4096, free), (free, 4096), ((1 << 16) + 1196, free), ((1 << 16) - 396, free), (free, (1 << 20) - 1196), (free, (1 << 21) + 296),
                       (free, (1 << 23) - 4)):
            assert call(g0, g1, bits) == -1, (bits, g0, g1)
    for g1 in ((1 << 24) - 4, 1 << 27):
        assert call(free, g1, 8) == -1
    assert call(free, free, 32, (1 << 16) + 1196) == -1
    assert call(free, free, 32, free) == -1


@pytest.mark.gpu
def test_a_callers_list_of_rates_may_change_between_steps(hip):
    p = [torch.ones(10, device=DEV), torch.ones(10, device=DEV)]
    z = lambda: [torch.zeros(10, device=DEV) for _ in p]
    plan = hip.adamw_plan(p, z(), z())
    lr, decay = [0.0, 0.5], [0.1, 0.1]
    plan.step(z(), 1, lr, B1, B2, EPS, decay)        # no gradient: p (1 - lr wd)
    lr[0], decay[1] = 0.5, 0.2
    plan.step(z(), 2, lr, B1, B2, EPS, decay)
    plan.step(z(), 3, np.float32(0.5), B1, B2, EPS, np.float64(0.5))
    for t, want in zip(p, (0.95 * 0.75, 0.95 * 0.9 * 0.75)):
        assert torch.allclose(t.cpu().double(), torch.full((10,), want, dtype=torch.float64), rtol=8 * U, atol=0)


@pytest.mark.gpu
def test_elements_past_31_bits(hip, monkeypatch):
    """A tensor of 2^31 + 700 elements, both its ends against the definition."""
    n, t, lr, wd = (1 << 31) + 700, 4, 1e-3, 0.01
    p = torch.full((n,), 0.25, dtype=torch.bfloat16, device=DEV)
    g = torch.full((n,), 1e-3, dtype=torch.bfloat16, device=DEV)
    code = lambda: torch.full((n,), 0x58, dtype=torch.uint8, device=DEV)
    scale = lambda: torch.full((-(-n // BLOCK),), 2.0 ** -10, device=DEV)
    m, v, ms, rs = code(), code(), scale(), scale()
    ends = [(0, 1000), ((1 << 31) - 512, n)]
    d = make(11, [hi - lo for lo, hi in ends], torch.bfloat16, torch.bfloat16, bits=8)
    for i, (lo, hi) in enumerate(ends):
        for whole, part in ((p, d["p"][i]), (g, d["g"][i]), (m, d["m"][i]), (v, d["v"][i])):
            whole[lo:hi] = part.to(DEV)
        for whole, part in ((ms, d["ms"][i]), (rs, d["rs"][i])):
            whole[lo // BLOCK:-(-hi // BLOCK)] = part.to(DEV)
    # the first range ends inside a block: the rest of that block is part of its scale
    ends[0], lo = (0, 768), 0
    f8 = lambda x: x.view(torch.float8_e4m3fn)
    hip.adamw([p], [g], [f8(m)], [f8(v)], t, lr, B1, B2, EPS, wd, scales=([ms], [rs]), seed=5)
    torch.cuda.synchronize()
    for i, (lo, hi) in enumerate(ends):
        k = hi - lo
        m0, r0 = values8(d["m"][i][:k], d["ms"][i][:-(-k // BLOCK)]), values8(d["v"][i][:k], d["rs"][i][:-(-k // BLOCK)])
        want, _, _, _, tol = step64(d["p"][i][:k], d["g"][i][:k], m0, r0 * r0, t, lr, wd)
        within(f"p from {lo}", p[lo:hi], want, tol + half_step(want.abs() + tol, torch.bfloat16))

        def bits_from(n, seed, step, index, lo=lo):
            h = _mix(torch.full((n,), _mix((seed + step * 0xA54FF53B + index * 0x3C6EF373) & M32), dtype=torch.int64) ^ (torch.arange(lo, lo + n) & M32))
            return h & 0xFFFF, h >> 16
        monkeypatch.setitem(globals(), "random_bits", bits_from)
        cm, cr, sm, sr = hold8(*states32(m0, r0 * r0, d["g"][i][:k].float()), 5, t, 0)
        assert torch.equal(m[lo:hi].cpu(), cm) and torch.equal(v[lo:hi].cpu(), cr)
        assert torch.equal(ms[lo // BLOCK:-(-hi // BLOCK)].cpu(), sm) and torch.equal(rs[lo // BLOCK:-(-hi // BLOCK)].cpu(), sr)
    monkeypatch.undo()
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("bits,pt,gt,n", [(32, "float32", "float32", 20_000_003), (8, "float32", "bfloat16", 40_000_001), (8, "bfloat16", "bfloat16", 60_000_003),
                                          (32, "float16", "float32", 26_000_000)])
def test_steps_past_the_caches_equal_small_ones(hip, bits, pt, gt, n):
    """A step of more than 384 MB reads and writes past the caches: bit for bit what its tensors' steps give in two parts.  (A
    tensor's random bits depend on its number in the list and the place in it: the parts keep both.)"""
    pt, gt = getattr(torch, pt), getattr(torch, gt)
    gen = torch.Generator(device=DEV).manual_seed(n)
    rnd = lambda n, dt, s: torch.randn(n, device=DEV, generator=gen).mul_(s).to(dt)
    sizes = [n, 5000, 255]

    def held(k):
        if bits == 32:
            return [torch.zeros(k, device=DEV), torch.zeros(k, device=DEV)], None
        return ([torch.zeros(k, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)],
                [torch.zeros(-(-k // BLOCK), device=DEV) for _ in range(2)])
    p, g = [rnd(k, pt, 0.1) for k in sizes], [rnd(k, gt, 1e-2) for k in sizes]
    whole, st = [t.clone() for t in p], [held(k) for k in sizes]
    for t in (1, 2):
        hip.adamw(whole, g, [s[0][0] for s in st], [s[0][1] for s in st], t, 1e-3, B1, B2, EPS, 0.01, seed=9,
                  scales=None if bits == 32 else ([s[1][0] for s in st], [s[1][1] for s in st]))
    half = n // 2 // 2048 * 2048
    # the same tensor's first part alone, in a list in which it has the same number and place
    part, sp = p[0][:half].clone(), held(half)
    for t in (1, 2):
        hip.adamw([part], [g[0][:half]], [sp[0][0]], [sp[0][1]], t, 1e-3, B1, B2, EPS, 0.01, seed=9,
                  scales=None if bits == 32 else ([sp[1][0]], [sp[1][1]]))
    raw = lambda t: t.view(torch.uint8)
    assert torch.equal(raw(whole[0][:half]), raw(part))
    assert all(torch.equal(raw(a[:half]), raw(b)) for a, b in zip(st[0][0], sp[0]))
    if bits == 8:
        assert all(torch.equal(a[:half // BLOCK], b) for a, b in zip(st[0][1], sp[1]))
    # its end against the definition (32 bits: no random bits in it)
    if bits == 32:
        e = slice(n - 5000, n)
        m = v = torch.zeros(5000)
        q = p[0][e].cpu()
        for t in (1, 2):
            want, _, _, _, tol = step64(q, g[0][e].cpu(), m, v, t, 1e-3, 0.01)
            m, v = states32(m, v, g[0][e].cpu().float())
            if t == 1:
                q = want.float().to(pt)
        within("m", st[0][0][0][e], m.double(), 4 * U * m.abs().double() + 1e-12)
        within("p", whole[0][e], want, 2 * tol + 3 * half_step(want.abs() + tol, pt))


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 1e-20])
def test_second_moments_among_the_denormals(hip, eps):
    """Gradients whose squares leave fp32's normal range, an epsilon that does not hide it.  p starts at zero, so that what is
    left is -size m / (sqrt(v) inv + eps) of the m and v that the GPU holds: 1 u each for size, its product, the root, inv, the
    denominator, eps and the result, 2 u for the reciprocal (one unit off at most): 9 u, 10 are used."""
    n, lr = 600, 1e-3
    g = torch.from_numpy(np.exp(np.random.default_rng(5).uniform(math.log(1e-20), math.log(1e-15), n)).astype(np.float32))
    g[::2] *= -1
    d = dict(p=[torch.zeros(n)], g=[g], m=[torch.zeros(n)], v=[torch.zeros(n)], ms=[], rs=[])
    gpu = {k: [t.to(DEV) for t in d[k]] for k in d}
    for t in (1, 2):
        gpu["p"][0].zero_()
        hip.adamw(gpu["p"], gpu["g"], gpu["m"], gpu["v"], t, lr, B1, B2, eps, 0.0)
        m, v = gpu["m"][0].cpu().double(), gpu["v"][0].cpu().double()
        assert bool((v > 0).all()) and bool((v < 2.0 ** -126).any()) and bool((v > 2.0 ** -126).any())
        # g^2, its product, v's product and their sum: half a denormal step each at most, and u of a normal one
        within("v", v, (1 - B2) * (1 + (t - 1) * B2) * g.double() ** 2, 5 * U * v + t * 2.0 ** -148)
        upd = lr / (1 - B1 ** t) * m / (v.sqrt() / math.sqrt(1 - B2 ** t) + eps)
        within("p", gpu["p"][0], -upd, 10 * U * upd.abs())


@pytest.mark.gpu
def test_8_bit_roots_of_second_moments_among_the_denormals(hip):
    """Blocks that hold nothing but such second moments: the codes are those of the format's definition, bit for bit."""
    sizes = [256, 700, 2048]
    rng = np.random.default_rng(9)
    d = dict(p=[], g=[], m=[], v=[], ms=[], rs=[])
    for n in sizes:
        d["p"].append(torch.zeros(n))
        d["g"].append(torch.from_numpy((rng.standard_normal(n) * 3e-19).astype(np.float32)))
        for k in ("m", "v"):
            d[k].append(torch.zeros(n, dtype=torch.uint8))
        for k in ("ms", "rs"):
            d[k].append(torch.zeros(-(-n // BLOCK)))
    got = run(hip, d, 8, 1, seed=17)
    for i, n in enumerate(sizes):
        cm, cr, ms, rs = hold8(*states32(torch.zeros(n), torch.zeros(n), d["g"][i]), 17, 1, i)
        assert torch.equal(got["ms"][i].cpu(), ms) and torch.equal(got["rs"][i].cpu(), rs)
        assert torch.equal(got["m"][i].cpu(), cm) and torch.equal(got["v"][i].cpu(), cr)
        assert len(set(cr.tolist())) > 20


def test_an_epsilon_among_the_denormals_is_refused():
    """(No GPU needed.)  The reciprocal takes such a denominator for zero: an element without a gradient would become NaN."""
    import pgan_hip
    from pgan_optim import AdamW
    P, LL, I, D = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_double
    one = lambda t, x: (t * 1)(x)
    for eps in (1e-45, 1e-39, 2.0 ** -127, math.inf * -1):
        assert pgan_hip._lib._real.pgan_adamw_multi(one(P, 4096), one(P, 1 << 16), one(P, 1 << 20), one(P, 1 << 21), None, None, one(LL, 100), one(I, 0),
                                                    one(D, 1e-3), one(D, 0.0), 1, 32, 0.5, 0.999, eps, 1.0, 0, None, 1, None) == -1
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(torch.zeros(3))], eps=eps)
    AdamW([torch.nn.Parameter(torch.zeros(3))], eps=2.0 ** -126)


@pytest.mark.gpu
def test_the_least_epsilon(hip):
    """Elements without a gradient stay where they are, at the smallest epsilon that is taken; at zero they are 0 / 0."""
    from pgan_hip import PganError
    g = torch.zeros(300, device=DEV)
    g[::3] = 1e-3
    for eps in (2.0 ** -126, 0.0):
        p, m, v = torch.ones(300, device=DEV), torch.zeros(300, device=DEV), torch.zeros(300, device=DEV)
        hip.adamw([p], [g], [m], [v], 1, 1e-3, B1, B2, eps, 0.0)
        still = p.cpu()[g.cpu() == 0]
        assert bool((still == 1).all()) if eps else bool(torch.isnan(still).all())
        within("p", p.cpu()[::3], torch.full((100,), 1 - 1e-3, dtype=torch.float64), torch.full((100,), 16 * U * 1e-3 + 4 * U, dtype=torch.float64))
    with pytest.raises(PganError):
        hip.adamw([p], [g], [m], [v], 1, 1e-3, B1, B2, 1e-39, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("b2,steps", [(0.9, 120), (0.99, 900)])
def test_the_8_bit_second_moment_over_many_steps(hip, b2, steps):
    """Gradients of variance 1: the mean V of the held root's square, which is what the next step starts from.  A rounding that is
    unbiased in the root adds its variance to the square, so V is no less than what 32 bits give, 1 - b2^t.  Nor is it much more:
    a rounded root stands on a code, the next step moves it by d = |sqrt(b2 r^2 + c2 g^2) - r| <= c2 |g^2 - r^2| / (2 r) (1 + c2),
    two neighbouring codes are at most s <= r / 8 apart, and rounding between them has a variance of at most d s, in the mean at
    most c2 (1 + c2) (1 + V) / 16.  With V = b2 V + c2 + that, k = (1 + c2) / 16: V <= (1 + k) / (1 - k), that is 1.16 for b2 =
    0.9 and 1.14 for 0.99.  Over n elements the mean is off by five times spread / sqrt(n) at most, a root that spreads by a
    half of itself and so a square by its whole included."""
    n = 1 << 16
    z = lambda k, dt: torch.zeros(k, dtype=dt, device=DEV)
    p, m, v, ms, rs = z(n, torch.float32), z(n, torch.uint8), z(n, torch.uint8), z(n // BLOCK, torch.float32), z(n // BLOCK, torch.float32)
    f8 = lambda x: x.view(torch.float8_e4m3fn)
    plan = hip.adamw_plan([p], [f8(m)], [f8(v)], scales=([ms], [rs]))
    gen = torch.Generator(device=DEV).manual_seed(8)
    for t in range(1, steps + 1):
        plan.step([torch.randn(n, device=DEV, generator=gen)], t, 1e-3, 0.9, b2, EPS, 0.0, seed=21)
    mean = float(values8(v.cpu(), rs.cpu()).double().square().mean())
    k, slack = (2 - b2) / 16, 5 / math.sqrt(n)
    print("second moment", mean)
    assert (1 - b2 ** steps) - slack <= mean <= (1 + k) / (1 - k) + slack
