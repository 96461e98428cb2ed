"""CPU-side checks of the drop-in surface: the C-ABI library loads and exports every symbol the
header declares, the nn.Module front-ends carry the reference's state_dict layout, the loaders and
the command line behave like the reference's (src/train_wgan_v2.py:227-351,372-430)."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import dcwgan_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    hdr = open(os.path.join(ROOT, "include", "pgan_hip.h")).read()
    declared = sorted(set(re.findall(r"\b(pgan_[a-z0-9_]+)\s*\(", hdr)))
    assert len(declared) >= 30
    lib = ctypes.CDLL(os.path.join(ROOT, "pg-alignments-gan_amd", "libpgan_hip.so"))
    for name in declared:
        assert hasattr(lib, name), f"{name} declared in include/pgan_hip.h but not exported"
    import pgan_hip
    assert sorted(pgan_hip.EXPORTS) == declared


def test_library_holds_no_packed_fp32_instructions(tmp_path):
    """Device code is built without the packed-fp32 vector instructions (v_pk_fma_f32, v_pk_mul_f32, v_pk_add_f32):
    kernels that held them returned wrong low halves of a register pair in one 16-lane row while kernels of other
    streams ran beside them.  Disassembles every gfx950 code object of the shipped library."""
    import shutil
    import subprocess
    objdump = "/opt/rocm/lib/llvm/bin/llvm-objdump"
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump")
    so = shutil.copy(os.path.join(ROOT, "pg-alignments-gan_amd", "libpgan_hip.so"), tmp_path / "lib.so")
    subprocess.run([objdump, "--offloading", str(so)], check=True, capture_output=True, cwd=tmp_path)
    objs = [f for f in os.listdir(tmp_path) if "gfx950" in f]
    assert len(objs) >= 8, objs
    kernels = 0
    for f in objs:
        asm = subprocess.run([objdump, "-d", str(tmp_path / f)], check=True, capture_output=True, text=True).stdout
        kernels += asm.count("s_endpgm")
        hits = re.findall(r"v_pk_(?:fma|mul|add)_f32", asm)
        assert not hits, f"{f}: {len(hits)} packed-fp32 instructions"
    assert kernels >= 50


def test_module_state_dict_layout_matches_reference_tables():
    import layers
    g = layers.DC_Generator_Leaky_Sig(64, 128, 0.1, 1, 4)
    d = layers.DC_Discriminator(64, 0.1, 1, 4)
    want_g = dict(orc.gen_param_shapes())
    want_g.update(orc.gen_buffer_shapes())
    got_g = {k: tuple(v.shape) for k, v in g.state_dict().items()}
    assert got_g == want_g
    assert {k: tuple(v.shape) for k, v in d.state_dict().items()} == orc.disc_param_shapes()
    assert g.state_dict()["twod_conv_layers.1.num_batches_tracked"].dtype == torch.int64
    assert sum(p.numel() for p in g.parameters()) == 3847824
    assert sum(p.numel() for p in d.parameters()) == 2777809
    # load_state_dict round trip keeps the flat backing store in sync
    sd = {k: torch.randn_like(v) if v.dtype == torch.float32 else v for k, v in d.state_dict().items()}
    d.load_state_dict(sd)
    assert torch.equal(d._store.p["out.weight"], sd["out.weight"])
    with pytest.raises(ValueError):
        layers.DC_Discriminator(128, 0.1, 1, 4)
    with pytest.raises(RuntimeError):
        d(torch.zeros(2, 1, 64, 64), torch.zeros(2, 1, 64))   # CPU tensors are rejected, no fallback


def _write_sims(tmp, n):
    rs, rp = orc.synthetic_alignments(n, 5)
    for i in range(n):
        np.savetxt(os.path.join(tmp, f"{i}_sites.csv"), rs[i, 0].numpy().astype(int), fmt="%d", delimiter=",")
        np.savetxt(os.path.join(tmp, f"{i}_pos.csv"), rp[i, 0].numpy(), fmt="%.6f")
    return rs, rp


def test_disk_loader(tmp_path):
    import train_wgan_v2 as tw
    rs, rp = _write_sims(str(tmp_path), 10)
    with pytest.raises(ValueError):
        tw.DataGeneratorDisk(str(tmp_path), num_in=11, batch_size=4)
    gen = tw.DataGeneratorDisk(str(tmp_path), num_in=10, batch_size=4)
    assert gen.length == 2
    s, p = gen.get_batch()
    assert tuple(s.shape) == (4, 1, 64, 64) and tuple(p.shape) == (4, 1, 64) and s.dtype == torch.float32
    sums = sorted(float(x.sum()) for x in rs)
    for x in s:
        assert any(abs(float(x.sum()) - v) < 1e-6 for v in sums)
    gen.get_batch()
    s3, p3 = gen.get_batch()                       # short last batch is returned as is
    assert s3.shape[0] == 2
    s4, _ = gen.get_batch()
    assert s4.shape[0] == 0
    gen.on_epoch_end()
    sh, _ = gen.get_batch(shuffle=True)            # rows permuted: column sums unchanged
    assert sh.shape[0] == 4
    alls, allp = gen.load_all()
    assert tuple(alls.shape) == (10, 1, 64, 64)
    assert abs(float(alls.sum()) - float(rs.sum())) < 1e-3
    assert torch.allclose(allp.sort(dim=0).values, rp.sort(dim=0).values, atol=1e-6)


def test_ms_parser_and_buffers():
    import train_wgan_v2 as tw
    rng = np.random.default_rng(0)
    lines = ["ms 64 3 -s 5", "1 2 3", ""]
    reps = []
    for r in range(3):
        pos = np.sort(rng.random(5))
        hap = rng.integers(0, 2, (64, 5))
        reps.append((pos, hap))
        lines += ["//", "segsites: 5", "positions: " + " ".join(f"{v:.4f}" for v in pos) + " "]
        lines += ["".join(str(c) for c in row) for row in hap] + [""]
    X, P = tw.read_ms_data(lines)
    assert X.shape == (2, 1, 64, 5) and P.shape == (2, 5, 1)     # last replicate dropped, as in the reference
    assert np.array_equal(X[1, 0], reps[1][1].astype(np.float32))
    assert np.allclose(P[0, :, 0], np.round(reps[0][0], 4), atol=1e-4)
    # the native parser (pgan_parse_ms) returns the same arrays, bit for bit
    Xn, Pn = tw.read_ms_text("\n".join(lines), rows=64, cols=5)
    assert Xn.shape == X.shape and Pn.shape == P.shape and np.array_equal(Xn, X) and np.array_equal(Pn, P)
    # a positions line without the trailing space loses its last value in the reference: 4 of 5 -> rejected
    broken = [ln.rstrip(" ") if ln.startswith("positions") else ln for ln in lines]
    assert tw.read_ms_data(broken)[1].shape == (2, 4, 1)
    with pytest.raises(ValueError):
        tw.read_ms_text("\n".join(broken), rows=64, cols=5)
    with pytest.raises(ValueError):
        tw.read_ms_text("\n".join(lines).replace("segsites: 5\n", "segsites: 5\nextra\n", 1), rows=64, cols=5)
    with pytest.raises(ValueError):
        tw.read_ms_text("\n".join(lines[:10] + ["0x010"] + lines[11:]), rows=64, cols=5)
    assert tw.read_ms_text("no replicates here\n")[0].shape[0] == 0
    buf = tw.FakeBuffer(max_size=8)
    buf.add(torch.arange(6).float().view(6, 1), torch.arange(6).float().view(6, 1))
    buf.add(torch.arange(6, 12).float().view(6, 1), torch.arange(6, 12).float().view(6, 1))
    assert buf.length == 8
    s, p = buf.sample(batch_size=8)
    assert sorted(s.flatten().tolist()) == [4, 5, 6, 7, 8, 9, 10, 11] and torch.equal(s, p)
    torch.manual_seed(0)
    probs = torch.full((3, 1, 64, 64), 1e-4)
    g = tw.sample_genotypes_bernoulli(probs)
    assert bool(((g.amax(dim=2) - g.amin(dim=2)) == 1).all())    # every column made polymorphic
    sites, pos = orc.synthetic_alignments(3, 1)
    s2, p2 = tw.switch_monomorphic(sites.clone(), pos.clone(), 4, 4)
    mono = ((s2.amax(dim=2) == s2.amin(dim=2))[:, 0]).sum(dim=1)
    assert mono.tolist() == [4, 4, 4]
    assert bool((p2[:, 0, 1:] >= p2[:, 0, :-1] - 1e-6).all())


def test_parse_args_flags(tmp_path):
    import train_wgan_v2 as tw
    od = tmp_path / "out"
    od.mkdir()
    (od / "stale.txt").write_text("x")
    a = tw.parse_args(["--odir", str(od), "--loss", "div", "--use_buffer", "--permute", "--normalize",
                       "--gen", "tanNorm", "--batch_size", "32"])
    assert a.loss == "div" and a.use_buffer and a.permute and a.normalize and a.gen == "tanNorm"
    assert a.batch_size == "32" and a.critic_iter == "5" and a.gp_lambda == "10" and a.gen_lr == "0.00005"
    assert list(od.iterdir()) == []            # an existing output directory is emptied, like the reference


def test_every_enqueue_entry_point_can_be_taped():
    """The native launch tape's registry (csrc/runtime.hip) knows every entry point that enqueues work, with the number
    of arguments the binding passes; host-side entry points cannot be noted."""
    import pgan_hip
    for name, kinds in pgan_hip._SIGS.items():
        if name in pgan_hip._Lib._HOST:
            assert pgan_hip._lib.pgan_tape_arg_count(name.encode()) == -1, name
        else:
            assert pgan_hip._lib.pgan_tape_arg_count(name.encode()) == len(kinds), name


def test_philox_words_known_answer():
    """The numpy restatement of the device generator (tests/torch_ops.py) reproduces the Random123 known answer of
    Philox4x32-10 (counter 0, key 0); the GPU tests hold the kernels to it word for word."""
    import torch_ops as T
    w = T.philox_words([0, 0, 0, 0], 0, 1)[0]
    assert [int(x) for x in w] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def test_library_states_its_build():
    import pgan_hip
    lib = ctypes.CDLL(pgan_hip.LIB_PATH)
    lib.pgan_build_info.restype = ctypes.c_char_p
    assert b"packed-fp32-ops=off" in lib.pgan_build_info()


def test_build_takes_its_former_argument():
    """build(force=True) and `__graft_entry__.py --force` (tools/ab_pk.sh): every call compiles everything either way."""
    import inspect
    import __graft_entry__ as entry
    inspect.signature(entry.build).bind()
    inspect.signature(entry.build).bind(True)
    inspect.signature(entry.build).bind(force=True)
