"""AdamW and the 8-bit sampler where a program uses them: the optimizer class on the drop-in modules, the fused trainer's
optimizer, alignments drawn from the generator that was trained, the command line.

Optimizer tolerances are those of test_adamw.step64, one step at a time from the states that the GPU held before it."""
import copy
import math
import os

import numpy as np
import pytest
import torch

import dcwgan_oracle as orc
from test_adamw import B1, B2, EPS, U, half_step, hold8, states32, step64, values8, within
from test_rows8 import codes_of, fold32, fold64, lrelu, same

DEV = torch.device("cuda:0")


def snapshot(opt, params):
    """Per parameter: value, first and second moment as fp32 values, steps made (None: no state yet)."""
    out = []
    for p in params:
        st = opt.state[p]
        if not st:
            out.append((p.detach().cpu().clone(), torch.zeros(p.numel()), torch.zeros(p.numel()), 0))
        elif "exp_avg_scale" in st:
            m = values8(st["exp_avg"].view(torch.uint8).cpu(), st["exp_avg_scale"].cpu())
            r = values8(st["exp_avg_sq"].view(torch.uint8).cpu(), st["exp_avg_sq_scale"].cpu())
            out.append((p.detach().cpu().clone(), m, r * r, st["step"]))
        else:
            out.append((p.detach().cpu().clone(), st["exp_avg"].cpu().clone(), st["exp_avg_sq"].cpu().clone(), st["step"]))
    return out


def check_step(before, params, grads, lr, wd, opt=None, bits=32):
    for i, ((p0, m0, v0, made), p, g) in enumerate(zip(before, params, grads)):
        if g is None:
            assert torch.equal(p.detach().cpu(), p0)
            continue
        want, mw, vw, terms, tol = step64(p0.reshape(-1), g.detach().cpu().reshape(-1), m0, v0, made + 1, lr, wd)
        within(f"p{i}", p.detach().reshape(-1), want, tol + half_step(want.abs() + tol, p.dtype))
        if opt is not None and bits == 32:
            within(f"m{i}", opt.state[p]["exp_avg"], mw, 4 * U * terms)
            within(f"v{i}", opt.state[p]["exp_avg_sq"], vw, 5 * U * vw)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_class(bits):
    """Two groups, parameters without a gradient in some steps, a gradient that is not contiguous, a learning rate that
    changes, five steps; then the same from a saved state, bit for bit."""
    from pgan_optim import AdamW
    gen = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.nn.Parameter(torch.randn(*s, generator=gen).to(DEV))
    a, b = [mk(33, 7), mk(300), mk(1)], [mk(64, 65), torch.nn.Parameter(torch.randn(500, generator=gen).to(DEV, torch.bfloat16))]
    opt = AdamW([dict(params=a, weight_decay=0.1), dict(params=b, lr=3e-3)], lr=1e-3, betas=(B1, B2), eps=EPS, weight_decay=0.0,
                state_bits=bits, seed=4)
    saved = None
    for k in range(5):
        grads = []
        for i, p in enumerate(a + b):
            g = torch.randn(*p.shape, generator=gen).to(DEV, p.dtype)
            if i == 3:
                g = torch.randn(65, 64, generator=gen).to(DEV).t()
            p.grad = None if i == 1 and k in (0, 3) else g
            grads.append(p.grad)
        if k == 3:
            saved, at = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in a + b]
            later = []
        if k == 2:
            for g in opt.param_groups:
                g["lr"] *= 0.5
        before = snapshot(opt, a + b)
        opt.step()
        torch.cuda.synchronize()
        check_step(before[:3], a, grads[:3], opt.param_groups[0]["lr"], 0.1, opt, bits)
        check_step(before[3:], b, grads[3:], opt.param_groups[1]["lr"], 0.0, opt, bits)
        if k >= 3:
            later.append([None if g is None else g.clone() for g in grads])
    assert [opt.state[p]["step"] for p in a + b] == [5, 3, 5, 5, 5]
    want = [p.detach().clone() for p in a + b]
    with torch.no_grad():
        for p, x in zip(a + b, at):
            p.copy_(x)
    again = AdamW([dict(params=a), dict(params=b)], state_bits=bits)
    again.load_state_dict(saved)
    for gs in later:
        for p, g in zip(a + b, gs):
            p.grad = g
        again.step()
    assert all(torch.equal(p.detach(), x) for p, x in zip(a + b, want))


@pytest.mark.gpu
def test_optimizer_takes_torchs_state_and_refuses_what_it_cannot_do():
    from pgan_hip import PganError
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.randn(40, 3, device=DEV))
    ref = torch.optim.AdamW([p], lr=1e-3, betas=(B1, B2), eps=EPS, weight_decay=0.02)
    for _ in range(2):
        p.grad = torch.randn(40, 3, device=DEV)
        ref.step()
    opt = AdamW([p])
    opt.load_state_dict(ref.state_dict())
    before = snapshot(opt, [p])
    assert before[0][3] == 2
    p.grad = torch.randn(40, 3, device=DEV)
    opt.step()
    check_step(before, [p], [p.grad], 1e-3, 0.02, opt)
    eight = AdamW([p], state_bits=8)
    with pytest.raises(ValueError):
        sd = ref.state_dict()
        sd["param_groups"][0]["state_bits"] = 8
        eight.load_state_dict(sd)
    had = snapshot(opt, [p])[0]
    with pytest.raises(ValueError):
        sd = ref.state_dict()
        del sd["state"][0]["exp_avg_sq"]
        opt.load_state_dict(sd)
    has = snapshot(opt, [p])[0]                      # as it was
    assert torch.equal(has[1], had[1]) and torch.equal(has[2], had[2]) and has[3] == had[3] == 3
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    cpu = torch.nn.Parameter(torch.zeros(3))
    cpu.grad = torch.zeros(3)
    with pytest.raises(RuntimeError):
        AdamW([cpu]).step()
    q = torch.nn.Parameter(torch.zeros(6, 4, device=DEV).t())
    q.grad = torch.zeros(6, 4, device=DEV).t()
    with pytest.raises(PganError):
        AdamW([q]).step()
    s = torch.nn.Parameter(torch.zeros(6, 4, device=DEV))
    s.grad = torch.zeros(6, 4, device=DEV).to_sparse()
    with pytest.raises(RuntimeError):
        AdamW([s]).step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_optimizer_step_counts_on_every_replay(bits):
    from pgan_optim import AdamW
    ps = [torch.nn.Parameter(torch.randn(n, device=DEV)) for n in (100, 700)]
    start = [p.detach().clone() for p in ps]
    gs = [[torch.randn(n, device=DEV) for n in (100, 700)] for _ in range(4)]
    for p in ps:
        p.grad = torch.zeros_like(p)
    load = lambda k: [p.grad.copy_(g) for p, g in zip(ps, gs[k])]
    opt = AdamW(ps, lr=1e-2, betas=(B1, B2), state_bits=bits, capturable=True)
    plain = AdamW(ps, lr=1e-2, betas=(B1, B2), state_bits=bits)
    graph = torch.cuda.CUDAGraph()
    load(0)
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            plain.step()
    opt.step()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 4):
        load(k)
        graph.replay()
        torch.cuda.synchronize()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [4, 4]
    got = [p.detach().clone() for p in ps]
    with torch.no_grad():
        for p, x in zip(ps, start):
            p.copy_(x)
    for k in range(4):
        load(k)
        plain.step()
    for p, x in zip(ps, got):        # the corrections pass through fp32 on the device: two roundings of each update
        assert float((p.detach() - x).abs().max()) <= 4 * (1e-2 * 4 * 8 * U + 4 * U * 5)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_drop_in_loop_with_adamw(bits):
    """The reference's critic statements with this optimizer in torch's place."""
    import layers
    from pgan_optim import AdamW
    torch.manual_seed(3)
    D = layers.DC_Discriminator(64, 0.1, 1, k_size=4).to(DEV)
    opt = AdamW(D.parameters(), lr=5e-5, betas=(B1, B2), weight_decay=0.01, state_bits=bits)
    rs, rp = orc.synthetic_alignments(8, 7)
    for _ in range(3):
        opt.zero_grad()
        loss = D(rs.to(DEV), rp.to(DEV)).mean()
        loss.backward()
        params = list(D.parameters())
        before = snapshot(opt, params)
        opt.step()
        check_step(before, params, [p.grad for p in params], 5e-5, 0.01, opt, bits)


def make_trainer(**kw):
    from pgan_hip import HipOps
    from pgan_trainer import FusedTrainer
    tr = FusedTrainer(HipOps(DEV, max_samples=64), 8, DEV, critic_iter=2, seed=77, **kw)
    gp_, dp = orc.make_params(orc.gen_param_shapes(), 5), orc.make_params(orc.disc_param_shapes(), 6)
    tr.eng.G.load(gp_)
    tr.eng.D.load(dp)
    tr.weights_changed()
    rs, rp = orc.synthetic_alignments(64, 9)
    tr.set_pool(rs, rp)
    return tr


def store_states(st, bits):
    if bits == 32:
        return {n: (st.m[n].reshape(-1).cpu().clone(), st.v[n].reshape(-1).cpu().clone()) for n in st.p}
    plan = st.adamw[0]
    out = {}
    for i, n in enumerate(st.p):
        m = values8(st.m[n].view(torch.uint8).cpu(), plan.scales[0][i].cpu())
        r = values8(st.v[n].view(torch.uint8).cpu(), plan.scales[1][i].cpu())
        out[n] = (m, r * r)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_steps_both_networks_with_adamw(bits):
    """Every parameter of both networks after an optimizer step of the engine; decay on weights only; the buffers between
    the parameters stay zero."""
    tr = make_trainer(optimizer="adamw", weight_decay=0.1, state_bits=bits)
    tr.iteration()
    e = tr.eng
    for st, lr, go in ((e.D, e.lr_d, e.adam_d), (e.G, e.lr_g, e.adam_g)):
        torch.cuda.synchronize()
        made = int(st.adamw[4][0])
        assert made == (2 if st is e.D else 1)
        before, held = {n: st.p[n].cpu().clone() for n in st.p}, store_states(st, bits)
        grads = {n: st.g[n].cpu().clone() for n in st.p}
        go()
        torch.cuda.synchronize()
        assert int(st.adamw[4][0]) == made + 1
        inside = torch.zeros(st.numel, dtype=torch.bool)
        for i, n in enumerate(st.p):
            m, v = held[n]
            wd = 0.1 if st.p[n].dim() > 1 else 0.0
            want, mw, vw, terms, tol = step64(before[n].reshape(-1), grads[n].reshape(-1), m, v, made + 1, lr, wd)
            # the corrections pass through fp32 on the device: 3 u more of the update, which 16 u of it covers
            within(n, st.p[n].reshape(-1), want, tol)
            if bits == 8:
                cm, cr, ms, rs = hold8(*states32(m, v, grads[n].reshape(-1)), 77 + (0 if st is e.D else 1), made + 1, i)
                assert torch.equal(st.m[n].view(torch.uint8).cpu(), cm) and torch.equal(st.v[n].view(torch.uint8).cpu(), cr)
            inside[st.offsets[n]:st.offsets[n] + st.p[n].numel()] = True
        assert bool((st.flat.cpu()[~inside] == 0).all())
    if bits == 8:
        assert e.D.mflat is None and e.G.vflat is None


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_on_a_tape_takes_the_eager_steps(bits):
    a, b = make_trainer(optimizer="adamw", state_bits=bits), make_trainer(optimizer="adamw", state_bits=bits)
    b.use_tape = True
    for _ in range(3):
        a.iteration()
        b.step()
    torch.cuda.synchronize()
    assert b.tape is not None
    for x, y in ((a.eng.D, b.eng.D), (a.eng.G, b.eng.G)):
        assert torch.equal(x.flat, y.flat)
        for n in x.p:
            assert torch.equal(x.m[n].view(torch.uint8), y.m[n].view(torch.uint8))
        assert torch.equal(x.adamw[4], y.adamw[4])


# ---- the sampler ---------------------------------------------------------------------------------------------------
def generator(seed, data=64):
    from pgan_engine import gen_buffer_shapes, gen_param_shapes
    P = {k: v.to(DEV) for k, v in orc.make_params(gen_param_shapes(128, data), seed).items()}
    rng = np.random.default_rng(seed)
    Bf = {}
    for k, s in gen_buffer_shapes(128, data).items():
        x = torch.from_numpy(rng.standard_normal(s).astype(np.float32))
        Bf[k] = (x * 0.2 if k.endswith("mean") else 0.3 + x.abs()).to(DEV)
    k = "twod_conv_layers.4.weight"
    P[k][3] = -P[k][3]              # a negative BatchNorm factor
    return P, Bf


def eval64(P, Bf, z, n, tower, act):
    """The generator in evaluation in 64 bits, and the standard deviation of what the 8-bit path adds to it when every rounding
    is independent and even over its step: a code's step is its row's scale (variance scale^2 / 12), for the tokens as for
    the channels; a tap in bf16 has a step of at most 2^-7 of its magnitude.  Variances pass a product with the squares of its
    other operand, a BatchNorm with the square of its factor, a LeakyReLU and the output with the square of their slope."""
    import torch.nn.functional as F
    d = lambda t: t.detach().cpu().double()
    x = d(z).view(z.shape[0], -1, 1, 1) if tower == "twod" else d(z).view(z.shape[0], -1, 1)
    var = torch.zeros_like(x)
    conv = F.conv_transpose2d if tower == "twod" else F.conv_transpose1d
    for i in range(n + 1):
        w = d(P[f"{tower}_conv_layers.{3 * i}.weight"])
        how = dict(stride=1) if i == 0 else dict(stride=2, padding=1)
        if tower == "twod":
            row = (x.abs().amax(1, keepdim=True) / 127).square() / 12
            col = (w.abs().amax(0, keepdim=True) / 127).square().expand_as(w) / 12
            var = conv(var + row, w.square(), **how) + conv(x.square(), col, **how)
            if i == 0:
                var = var + (2.0 ** -7 * conv(x, w, **how)).square() / 12
            else:                                        # a pixel's four taps
                taps = sum(conv(x, w * sel, **how).square() for sel in tap_masks(w))
                var = var + 2.0 ** -14 * taps / 12
        x = conv(x, w, **how)
        if i < n:
            k = f"{tower}_conv_layers.{3 * i + 1}"
            gain = d(P[k + ".weight"]) / torch.sqrt(d(Bf[k + ".running_var"]) + 1e-5)
            shape = (1, -1) + (1,) * (x.dim() - 2)
            x = (x - d(Bf[k + ".running_mean"]).view(shape)) * gain.view(shape) + d(P[k + ".bias"]).view(shape)
            if tower == "twod":
                var = var * gain.square().view(shape) * torch.where(x > 0, 1.0, 0.01)
            x = torch.where(x > 0, x, 0.1 * x)
    out = torch.sigmoid(x) if act == "sigmoid" else torch.tanh(x)
    slope = out * (1 - out) if act == "sigmoid" else 1 - out * out
    return out, (var.sqrt() * slope + 1e-6) if tower == "twod" else None


def tap_masks(w):
    """One mask of the 4 x 4 kernel for each of the four taps that an output pixel takes: (0 or 1, or 2 or 3) each way."""
    out = []
    for a in (slice(0, 2), slice(2, 4)):
        for b in (slice(0, 2), slice(2, 4)):
            m = torch.zeros(4, 4, dtype=w.dtype)
            m[a, b] = 1
            out.append(m)
    return out


def near(got, want, sigma):
    """Within the roundings' spread: no value further off than eight standard deviations, and on average (in squares) no more
    than twice what independent roundings give -- a scale, tap or channel in the wrong place is off by whole values."""
    off = (got.double().cpu() - want).abs()
    print("largest error", float(off.max()), "rms", float(off.square().mean().sqrt()), "expected", float(sigma.square().mean().sqrt()))
    assert bool((off <= 8 * sigma).all())
    assert float(off.square().mean()) <= 4 * float(sigma.square().mean())


@pytest.mark.gpu
@pytest.mark.parametrize("data,act,n", [(64, "sigmoid", 1), (64, "tanh", 5), (128, "sigmoid", 3), (64, "sigmoid", 40)])
def test_sampler_stage_by_stage(data, act, n):
    """Each product and fold of a draw from the codes and taps that the GPU held before it; the drawn sites within the
    spread of the roundings; the positions in fp32."""
    from pgan_hip import HipOps
    from pgan_sampler import Sampler8
    hip = HipOps(DEV, max_samples=64)
    P, Bf = generator(3, data)
    s = Sampler8(hip, P, Bf, 40, act, 128, data)
    z = torch.randn(n, 128, generator=torch.Generator().manual_seed(n)).to(DEV)
    sites, pos = s.draw(z)
    torch.cuda.synchronize()
    assert tuple(sites.shape) == (n, 1, data, data) and tuple(pos.shape) == (n, 1, data)
    for i in range(1, s.n + 1):
        px, c, h = n * s.g2h[i] ** 2, s.g2c[i], s.g2h[i]
        y = s.y[i][:px].cpu()
        q, qs, w, ws = s.q[i][:px].cpu(), s.qs[i][:px].cpu(), s.w[i].cpu(), s.ws[i].cpu()
        rows = torch.randperm(px, generator=torch.Generator().manual_seed(1))[:200]
        want = (q[rows].double() @ w.double().t()) * (qs[rows].double()[:, None] * ws.double()[None])
        assert bool(((y[rows].double() - want).abs() <= (4 * U + 2.0 ** -8) * want.abs() * (1 + 2.0 ** -7)).all())
        few = min(n, 3)
        taps = y.view(n, h, h, -1)[:few]
        if i < s.n:
            cq, cs = codes_of(lrelu(fold32(taps, s.shift[i].cpu())).reshape(-1, s.g2c[i + 1]))
            m = few * 4 * h * h
            assert torch.equal(s.q[i + 1][:m].cpu(), cq)
            same(s.qs[i + 1][:m].cpu(), cs)
        else:
            o, tol = fold64(taps, None)
            o = torch.sigmoid(o) if act == "sigmoid" else torch.tanh(o)
            assert bool(((sites[:few].permute(0, 2, 3, 1).double().cpu() - o).abs() <= tol + 8 * U).all())
    cq, cs = codes_of(lrelu(s.y[0][:n].cpu().float()).view(-1, s.g2c[1]))
    assert torch.equal(s.q[1][:n * 16].cpu(), cq)
    same(s.qs[1][:n * 16].cpu(), cs)
    near(sites, *eval64(P, Bf, z, s.n, "twod", act))
    want, _ = eval64(P, Bf, z, s.n, "oned", act)
    assert float((pos.double().cpu() - want).abs().max()) <= 1e-5
    alone, _ = s.draw(z[:1])                         # an alignment does not depend on what it is drawn beside
    assert torch.equal(alone[0].clone(), s.draw(z)[0][0])


@pytest.mark.gpu
def test_sampler_refusals_and_refresh():
    from pgan_hip import HipOps, PganError
    from pgan_sampler import Sampler8
    hip = HipOps(DEV, max_samples=64)
    P, Bf = generator(8)
    with pytest.raises(ValueError):
        Sampler8(hip, P, Bf, 0)
    with pytest.raises(ValueError):
        Sampler8(hip, P, Bf, 4, act="relu")
    s = Sampler8(hip, P, Bf, 4)
    for bad in (torch.zeros(5, 128, device=DEV), torch.zeros(2, 64, device=DEV)):
        with pytest.raises(PganError):
            s.draw(bad)
    assert s.draw(torch.zeros(0, 128, device=DEV))[0].shape == (0, 1, 64, 64)
    z = torch.randn(4, 128, 1, 1, device=DEV)
    first = s.draw(z)[0].clone()
    P["twod_conv_layers.3.weight"].mul_(1.5)
    Bf["oned_conv_layers.1.running_mean"].add_(0.3)
    was = s.draw(z)
    assert torch.equal(was[0], first)
    p0 = was[1].clone()
    s.refresh()
    now = s.draw(z)
    assert not torch.equal(now[0], first) and not torch.equal(now[1], p0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.draw(z)
    want = [t.clone() for t in s.draw(z)]
    for _ in range(3):
        s.draw(torch.zeros_like(z))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s.sites.view(4, 1, 64, 64), want[0]) and torch.equal(s.pos, want[1])
    with pytest.raises(PganError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            s.draw(z[:3])


@pytest.mark.gpu
def test_train_then_draw():
    """The operators together: both networks trained with AdamW in 8 bits, then alignments drawn from the generator."""
    tr = make_trainer(optimizer="adamw", state_bits=8, lr_g=1e-3)
    for _ in range(3):
        tr.step()
    s = tr.sampler8(16)
    z = torch.randn(16, 128, device=DEV)
    sites, pos = s.draw(z)
    near(sites, *eval64(tr.eng.G.p, tr.eng.Gbuf.p, z, s.n, "twod", "sigmoid"))
    import train_wgan_v2 as tw
    bits, p = tw.draw_alignments(tr, 37, False, batch=16)
    assert bits.shape == (37, 512) and bits.dtype == np.uint8 and p.shape == (37, 64) and p.dtype == np.float32
    assert bool(np.isfinite(p).all()) and 0 < np.unpackbits(bits).mean() < 1


@pytest.mark.gpu
def test_module_sampler():
    import layers
    torch.manual_seed(1)
    G = layers.DC_Generator_Leaky_Tan(64, 128, 0.1, 1, k_size=4)
    with pytest.raises(RuntimeError):
        G.sampler8(2)
    G = G.to(DEV)
    G(torch.randn(8, 128, 1, 1, device=DEV))         # running statistics
    s = G.sampler8(4)
    z = torch.randn(3, 128, 1, 1, device=DEV)
    sites, _ = s.draw(z)
    near(sites, *eval64(G._store.p, G._bstore.p, z, s.n, "twod", "tanh"))


@pytest.mark.gpu
def test_command_line(tmp_path):
    import alignment_slab
    import train_wgan_v2 as tw
    from test_hip_cli import _write_sims
    idir, odir, slab = tmp_path / "sims", tmp_path / "out", tmp_path / "drawn.slab"
    idir.mkdir()
    _write_sims(str(idir), 96)
    tw.main(["--idir", str(idir), "--odir", str(odir), "--use_cuda", "--num_in", "96", "--batch_size", "8", "--epochs", "1",
             "--save_freq", "1", "--optimizer", "adamw", "--weight_decay", "0.02", "--state_bits", "8", "--draw_n", "300",
             "--draw_slab", str(slab)])
    g = torch.load(odir / "generator_model_0001.pt", weights_only=True)
    assert all(bool(torch.isfinite(v.float()).all()) for v in g.values())
    bits, pos = alignment_slab.read_slab(str(slab))
    assert bits.shape == (300, 512) and pos.shape == (300, 64)
    base = ["--idir", str(idir), "--odir", str(odir), "--use_cuda", "--num_in", "96", "--batch_size", "8", "--epochs", "1"]
    for bad in (["--optimizer", "sgd"], ["--state_bits", "16"], ["--draw_n", "3"], ["--draw_slab", "x"]):
        with pytest.raises(SystemExit):
            tw.main(base + bad)


def test_adamw_needs_the_gpu_backend():
    from pgan_trainer import FusedTrainer
    from torch_ops import TorchOps
    with pytest.raises(RuntimeError):
        FusedTrainer(TorchOps(), 4, torch.device("cpu"), optimizer="adamw")
    with pytest.raises(ValueError):
        FusedTrainer(TorchOps(), 4, torch.device("cpu"), optimizer="sgd")
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError):
        AdamW([p]).step()


@pytest.mark.gpu
def test_optimizer_follows_its_parameters_and_counter():
    from pgan_hip import PganError
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.randn(6, 4, device=DEV))
    opt = AdamW([p], capturable=True)
    p.grad = torch.ones_like(p)
    opt.step()
    late = AdamW([p], weight_decay=0.0)
    late.step()
    late.param_groups[0]["capturable"] = True        # the counter on the device is made by the next eager step
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            late.step()
    late.step()
    assert int(late.param_groups[0]["counter"][0]) == 2
    p.data = p.data.t()                              # the same memory in another order
    p.grad = torch.ones_like(p)
    with pytest.raises(PganError):
        opt.step()


@pytest.mark.gpu
def test_engine_adamw_refusals_and_late_start():
    from pgan_hip import HipOps
    from pgan_trainer import FusedTrainer
    tr = FusedTrainer(HipOps(torch.device(DEV)), 8, DEV, critic_iter=1)
    for bad in (dict(weight_decay=-1.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            tr.eng.use_adamw(**bad)
    tr.eng.D.step = tr.eng.G.step = 7                # as after seven steps of Adam
    tr.eng.use_adamw(0.0)
    assert int(tr.eng.D.adamw[4][0]) == 7            # goes on with Adam's moments
    tr.eng.use_adamw(0.0, state_bits=8)
    assert int(tr.eng.D.adamw[4][0]) == 0            # moments of zero are those of no step
    with pytest.raises(RuntimeError):
        tr.eng.use_adamw(0.0, state_bits=32)


@pytest.mark.gpu
def test_draw_slab_needs_its_folder(tmp_path):
    import train_wgan_v2
    with pytest.raises(SystemExit, match="no folder"):
        train_wgan_v2.main(["--use_cuda", "--idir", str(tmp_path), "--odir", str(tmp_path), "--draw_n", "4", "--draw_slab", str(tmp_path / "none" / "x.slab")])


@pytest.mark.gpu
def test_a_captured_draw_follows_refresh():
    """Weights and statistics change under a sampler: draws stay those of the last refresh(), a captured one's replays too."""
    from pgan_hip import HipOps
    from pgan_sampler import Sampler8
    P, Bf = generator(21)
    s = Sampler8(HipOps(DEV, max_samples=8), P, Bf, 8)
    z = torch.randn(4, 128, device=DEV)
    first = [t.clone() for t in s.draw(z)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.draw(z)
    gen = torch.Generator(device=DEV).manual_seed(3)
    for t in list(P.values()) + [v for k, v in Bf.items() if "running" in k]:
        t.mul_(1 + 0.2 * torch.rand(t.shape, device=DEV, generator=gen))
    assert all(torch.equal(a, b) for a, b in zip(s.draw(z), first))
    graph.replay()
    assert torch.equal(s.pos[:4], first[1])
    s.refresh()
    keep = [torch.full((1 << 16,), float("nan"), device=DEV) for _ in range(64)]      # what a freed buffer would hold
    for _ in range(3):
        s.draw(torch.zeros_like(z))
        graph.replay()
        torch.cuda.synchronize()
        got = s.sites[:4].clone(), s.pos[:4].clone()
        want = s.draw(z)
        assert torch.equal(got[0].view(4, 1, 64, 64), want[0]) and torch.equal(got[1], want[1])
        assert not torch.equal(want[0], first[0]) and not torch.equal(want[1], first[1])
    near(want[0], *eval64(P, Bf, z, s.n, "twod", "sigmoid"))
    pos, _ = eval64(P, Bf, z, s.n, "oned", "sigmoid")
    assert float((want[1].double().cpu() - pos).abs().max()) < 1e-4
    del keep


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_in_a_graph_takes_the_eager_steps(bits):
    a, b = make_trainer(optimizer="adamw", state_bits=bits), make_trainer(optimizer="adamw", state_bits=bits)
    b.capture()                                      # makes one iteration
    a.iteration()
    for _ in range(3):
        a.iteration()
        b.replay()
    torch.cuda.synchronize()
    for x, y in ((a.eng.D, b.eng.D), (a.eng.G, b.eng.G)):
        assert torch.equal(x.flat, y.flat) and torch.equal(x.adamw[4], y.adamw[4])
        for n in x.p:
            assert torch.equal(x.m[n].view(torch.uint8), y.m[n].view(torch.uint8))
            assert torch.equal(x.v[n].view(torch.uint8), y.v[n].view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_follows_load_state_dict(bits):
    from pgan_optim import AdamW
    torch.manual_seed(4)
    start = torch.randn(700, device=DEV)
    grads = [torch.randn(700, device=DEV) for _ in range(6)]

    def run(captured):
        p = torch.nn.Parameter(start.clone())
        p.grad = torch.zeros_like(p)
        opt = AdamW([p], lr=1e-2, betas=(B1, B2), eps=EPS, state_bits=bits, seed=3, capturable=True)

        def step(g, how):
            p.grad.copy_(g)
            how()
        step(grads[0], opt.step)
        step(grads[1], opt.step)
        saved, at = copy.deepcopy(opt.state_dict()), p.detach().clone()
        how = opt.step
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
            how = graph.replay
        step(grads[2], how)
        step(grads[3], how)
        mid = p.detach().clone()
        p.data.copy_(at)
        opt.load_state_dict(saved)
        junk = [torch.full((700,), float("nan"), device=DEV) for _ in range(16)]
        step(grads[4], how)
        step(grads[5], how)
        torch.cuda.synchronize()
        del junk
        assert opt.state_dict()["state"][0]["step"] == 4
        return [mid, p.detach().clone()] + [t.view(torch.uint8) for k, t in opt.state[p].items() if k != "step"]
    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_backward_pass_over_stepped_weights_is_refused():
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.randn(30, device=DEV))
    opt = AdamW([p])
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Each operator on two streams beside each other, with buffers of their own, gives what it gives alone."""
    from pgan_hip import HipOps, rows8
    hip = HipOps(DEV, ws_floats=4, max_samples=1)
    gen = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=gen)

    def lane(T, K, N, n):
        x, w, ws, y = rnd(T, K).bfloat16(), rows8(N, K, DEV), torch.zeros(N, device=DEV), torch.zeros(T, N, device=DEV)
        hip.quant_rows(rnd(N, K), w, ws)
        q, qs, taps = rows8(T, K, DEV), torch.zeros(T, device=DEV), rnd(n, 6, 6, 16 * 24).half()
        fq, fs = rows8(n * 144, 24, DEV), torch.zeros(n * 144, device=DEV)
        p, g = [rnd(n * 1000), rnd(300)], [rnd(n * 1000), rnd(300)]
        m, v = ([torch.zeros(t.numel(), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for t in p] for _ in range(2))
        sc = [[torch.zeros(-(-t.numel() // 256), device=DEV) for t in p] for _ in range(2)]
        start = [t.clone() for t in p]
        plan = hip.adamw_plan(p, m, v, sc)

        def reset():
            for t, s in zip(p, start):
                t.copy_(s)
            for t in m + v + sc[0] + sc[1] + [y, fs]:
                t.view(torch.uint8).zero_()

        def work():
            for t in range(1, 9):
                hip.linear_q8(x, w, ws, y, q, qs, lrelu=True)
                plan.step(g, t, 1e-2, B1, B2, EPS, 0.01, seed=4)
                hip.up_fold_q8(taps, None, fq, fs)
        results = lambda: [t.view(torch.uint8).clone() for t in [y, fq.contiguous(), fs] + p + m + v + sc[0] + sc[1]]
        return reset, work, results
    lanes = [lane(700, 640, 900, 40), lane(20, 300, 70, 7)]
    want = []
    for reset, work, results in lanes:
        reset()
        work()
        torch.cuda.synchronize()
        want.append(results())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for reset, _, _ in lanes:
            reset()
        torch.cuda.synchronize()
        for s, (_, work, _) in zip(streams, lanes):
            with torch.cuda.stream(s):
                work()
        torch.cuda.synchronize()
        for (_, _, results), w in zip(lanes, want):
            assert all(torch.equal(a, b) for a, b in zip(results(), w))


@pytest.mark.gpu
@pytest.mark.parametrize("latent,n", [(1024, 12), (1024, 16), (1024, 8), (512, 16), (2048, 7), (16, 3)])
def test_sampler_of_other_latent_sizes(latent, n):
    """Draws of a few alignments from latent vectors of any multiple of 16: the first product from its definition, the sites
    within the spread of the roundings."""
    from pgan_engine import gen_buffer_shapes, gen_param_shapes
    from pgan_hip import HipOps
    from pgan_sampler import Sampler8
    P = {k: v.to(DEV) for k, v in orc.make_params(gen_param_shapes(latent, 64), 31).items()}
    rng = np.random.default_rng(31)
    Bf = {}
    for k, shape in gen_buffer_shapes(latent, 64).items():
        x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32))
        Bf[k] = (x * 0.2 if k.endswith("mean") else 0.3 + x.abs()).to(DEV)
    s = Sampler8(HipOps(DEV, max_samples=64), P, Bf, n, "sigmoid", latent)
    z = torch.randn(n, latent, generator=torch.Generator().manual_seed(n))
    sites, pos = s.draw(z.to(DEV))
    q, qs = codes_of(z)
    want = (q.double() @ s.w[0].cpu().double().t()) * (qs.double()[:, None] * s.ws[0].cpu().double()) + s.bias0.cpu().double()
    tol = 4 * U * (want.abs() + 2 * s.bias0.cpu().double().abs())
    within("y0", s.y[0][:n], want, tol + half_step(want.abs() + tol, torch.bfloat16))
    near(sites, *eval64(P, Bf, z, s.n, "twod", "sigmoid"))
    assert bool(torch.isfinite(pos).all())


@pytest.mark.parametrize("other,options", [("AdamW", dict(maximize=True)), ("AdamW", dict(amsgrad=True)), ("AdamW", dict(differentiable=True)),
                                           ("Adam", dict(weight_decay=0.1)), ("Adam", dict(maximize=True))])
def test_options_that_a_step_would_pass_over_are_refused(other, options):
    """A state of torch's whose step would be another one here; nothing changes.  (No GPU needed.)"""
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.ones(5))
    p.grad = torch.ones(5)
    ref = getattr(torch.optim, other)([p], lr=0.125, **options)
    if not options.get("differentiable"):
        ref.step()
    opt = AdamW([p], lr=0.25)
    with pytest.raises(ValueError):
        opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.25 and len(opt.state) == 0 and "maximize" not in opt.param_groups[0]
    if other == "AdamW":
        with pytest.raises(ValueError):
            AdamW([dict(params=[p], **options)])


def test_states_of_adam_without_a_decay_are_taken():
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.ones(5))
    p.grad = torch.ones(5)
    ref = torch.optim.Adam([p], lr=0.125)
    ref.step()
    opt = AdamW([p])
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.125 and opt.state[p]["step"] == 1 and torch.equal(opt.state[p]["exp_avg"], ref.state[p]["exp_avg"])


def test_a_decay_given_after_adams_states_were_taken():
    """Its own saved state goes back in.  (No GPU needed.)"""
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.ones(5))
    p.grad = torch.ones(5)
    ref = torch.optim.Adam([p], lr=0.125)
    ref.step()
    opt = AdamW([p])
    opt.load_state_dict(ref.state_dict())
    opt.param_groups[0]["weight_decay"] = 0.25
    again = AdamW([p])
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[0]["weight_decay"] == 0.25


def test_load_hooks_see_and_may_change_the_states():
    """torch's hooks around load_state_dict: the one before gets the saved states and what it makes of them is loaded, the one
    after finds them in place.  (No GPU needed.)"""
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.ones(5))
    p.grad = torch.ones(5)
    ref = torch.optim.AdamW([p], lr=0.125)
    ref.step()
    opt, seen = AdamW([p]), []

    def before(o, sd):
        seen.append(sorted(sd["state"][0]))
        st = {0: {**sd["state"][0], "exp_avg": sd["state"][0]["exp_avg"] * 2}}
        return {**sd, "state": st}

    def after(o):
        seen.append((o.state[p]["step"], o.state[p]["exp_avg"].clone()))
    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(after)
    saved = ref.state_dict()
    opt.load_state_dict(saved)
    opt.load_state_dict(saved)                       # once each time
    assert seen[0] == seen[2] == ["exp_avg", "exp_avg_sq", "step"] and seen[1][0] == 1 and len(seen) == 4
    assert torch.equal(seen[1][1], 2 * ref.state[p]["exp_avg"]) and torch.equal(opt.state[p]["exp_avg"], 2 * ref.state[p]["exp_avg"])
    with pytest.raises(ValueError):                  # a hook's states are checked as any
        bad = AdamW([p])
        bad.register_load_state_dict_pre_hook(lambda o, sd: {**sd, "state": {0: {"step": 1}}})
        bad.load_state_dict(saved)
    assert len(bad.state) == 0


def test_groups_keep_options_that_a_loaded_state_does_not_name():
    """torch's states know neither bits nor seeds: each group's own stay, not the constructor's.  (No GPU needed.)"""
    from pgan_optim import AdamW
    a, b = torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(6))
    a.grad, b.grad = torch.ones(5), torch.ones(6)
    ref = torch.optim.AdamW([dict(params=[a]), dict(params=[b])], lr=0.125)
    ref.step()
    opt = AdamW([dict(params=[a], seed=5), dict(params=[b])], seed=9)
    opt.load_state_dict(ref.state_dict())
    assert [g["seed"] for g in opt.param_groups] == [5, 9] and [g["lr"] for g in opt.param_groups] == [0.125, 0.125]
    opt = AdamW([dict(params=[a], state_bits=8), dict(params=[b])])
    with pytest.raises(ValueError):                  # states of 32 bits for a group that holds 8
        opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["state_bits"] == 8
    opt = AdamW([dict(params=[a], state_bits=32), dict(params=[b], state_bits=32)], state_bits=8)
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["state_bits"] == 32 and opt.state[a]["exp_avg"].dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_after_loading_a_state_that_is_not_capturable(bits):
    """Its counter and states stay allocated, and it counts on from what was loaded: replays equal numbered steps, and what is
    allocated after the load is left alone."""
    from pgan_optim import AdamW
    torch.manual_seed(6)
    start = torch.randn(700, device=DEV)
    grads = [torch.randn(700, device=DEV) for _ in range(6)]
    p = torch.nn.Parameter(start.clone())
    p.grad = torch.zeros_like(p)
    kw = dict(lr=1e-2, betas=(B1, B2), eps=EPS, state_bits=bits, seed=3)
    plain = AdamW([p], **kw)
    for g in grads[:3]:
        p.grad.copy_(g)
        plain.step()
    saved, at = copy.deepcopy(plain.state_dict()), p.detach().clone()
    for g in grads[3:5]:
        p.grad.copy_(g)
        plain.step()
    want = [p.detach().clone()] + [t.clone() for k, t in plain.state[p].items() if k != "step"]
    p.data.copy_(start)
    opt = AdamW([p], capturable=True, **kw)
    p.grad.copy_(grads[0])
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(saved)
    assert not opt.param_groups[0]["capturable"]
    p.data.copy_(at)
    torch.cuda.synchronize()
    junk = [torch.full((4,), 7, dtype=torch.int32, device=DEV) for _ in range(512)] + [torch.full((700,), 7, dtype=torch.int32, device=DEV) for _ in range(32)]
    for g in grads[3:5]:
        p.grad.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in junk)
    got = [p.detach()] + [t for k, t in opt.state[p].items() if k != "step"]
    if bits == 8:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[1:], want[1:]))
    # the corrections pass through fp32 on the device: two roundings of each update, |update| < 8 lr here
    assert float((got[0] - want[0]).abs().max()) <= 2 * (1e-2 * 8 * 8 * U + 4 * U * 5)


@pytest.mark.gpu
def test_states_of_a_captured_step_stay_allocated():
    """A load that brings no states takes the optimizer's away, not the memory that the captured step writes to."""
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.randn(900, device=DEV))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], capturable=True)
    none = copy.deepcopy(opt.state_dict())
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(none)
    assert len(opt.state) == 0
    torch.cuda.synchronize()
    junk = [torch.full((900,), 7, dtype=torch.int32, device=DEV) for _ in range(64)] + [torch.full((4,), 7, dtype=torch.int32, device=DEV) for _ in range(512)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in junk)
    opt.step()                                       # starts anew
    assert int(opt.param_groups[0]["counter"][0]) == 1


@pytest.mark.gpu
def test_a_group_that_stops_counting_on_the_device():
    """The steps made so far count on, in numbered steps and, after another change, on the device again."""
    from pgan_optim import AdamW
    p = torch.nn.Parameter(torch.randn(300, device=DEV))
    opt = AdamW([p], lr=1e-2, betas=(B1, B2), eps=EPS, weight_decay=0.0, capturable=True)
    for k in range(6):
        opt.param_groups[0]["capturable"] = k not in (3, 4)
        p.grad = torch.randn(300, device=DEV)
        m, v = (opt.state[p][n].cpu().clone() if k else torch.zeros(300) for n in ("exp_avg", "exp_avg_sq"))
        p0 = p.detach().cpu().clone()
        opt.step()
        want, _, _, _, tol = step64(p0, p.grad.cpu(), m, v, k + 1, 1e-2, 0.0)
        within(f"step {k + 1}", p.detach(), want, tol)
    assert opt.state_dict()["state"][0]["step"] == 6


@pytest.mark.gpu
def test_drawn_alignments_follow_the_runs_seed():
    """Whatever the global generator went through before; a second draw of the same trainer is another one."""
    import train_wgan_v2 as tw

    def draws(seed, before):
        tr = make_trainer()
        tr.seed = seed
        tw.set_genotype_sampler(tr.ops, seed + 6)
        torch.manual_seed(before)
        torch.randn(before, device=DEV)
        first = tw.draw_alignments(tr, 21, False, batch=8)
        torch.manual_seed(before)
        return first, tw.draw_alignments(tr, 21, False, batch=8)
    try:
        a, b, c = draws(77, 5), draws(77, 900), draws(78, 5)
    finally:
        tw._GENOTYPE_RNG.clear()
    for x, y in zip(a, b):
        assert np.array_equal(x[0], y[0]) and np.array_equal(x[1], y[1])
    assert not np.array_equal(a[0][1], a[1][1]) and not np.array_equal(a[0][1], c[0][1])
