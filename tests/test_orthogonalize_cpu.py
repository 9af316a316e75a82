"""Argument checks of cfp_orthogonalize / cfp_muon_update: every refusal comes before the first
HIP call, so none of this needs a GPU."""
import ctypes as C

import pytest

P = C.c_void_p(0x10000)   # never dereferenced: each call below is refused on the host
BIG = 1 << 40


def _ortho(lib, g=P, dtype=0, ld=64, stride=64 * 64, batch=1, rows=64, cols=64, steps=5, eps=1e-7, products=0, out=P,
           ldo=64, so=64 * 64, work=P, nbytes=BIG):
    return lib.cfp_orthogonalize(g, dtype, ld, stride, batch, rows, cols, steps, None, eps, products, out, ldo, so,
                                 work, nbytes, None)


def _muon(lib, w=P, g=P, m=P, ld=64, stride=64 * 64, batch=1, rows=64, cols=64, steps=5, products=0, work=P, nbytes=BIG,
          eps=1e-7):
    return lib.cfp_muon_update(w, g, m, ld, stride, batch, rows, cols, None, 0.1, 0.9, 1, 0.0, 0.0, steps, None, eps,
                               products, work, nbytes, None)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=3), "dtype"), (dict(batch=-1), "batch"), (dict(batch=65536), "batch"), (dict(rows=0), "rows"),
    (dict(cols=65537, ld=65537), "cols"), (dict(steps=17), "steps"), (dict(steps=-1), "steps"),
    (dict(products=2), "products"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(g=None), "NULL"),
    (dict(out=None), "NULL"), (dict(ld=63), "strides"), (dict(ldo=63), "strides"),
    (dict(batch=2, stride=64 * 64 - 1), "overlap"), (dict(batch=2, so=0), "overlap"),
    (dict(g=C.c_void_p(0x10002)), "aligned"), (dict(dtype=1, out=C.c_void_p(0x10001)), "aligned"),
    (dict(work=None, rows=300), "workspace"), (dict(nbytes=1000, rows=300), "workspace"),
    (dict(work=C.c_void_p(0x10010), rows=300), "workspace"),
])
def test_orthogonalize_refuses(pkg, kw, word):
    lib = pkg.lib()
    assert _ortho(lib, **kw) != 0
    assert word in lib.cfp_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(w=None), "NULL"), (dict(g=None), "NULL"), (dict(m=None), "NULL"), (dict(ld=10), "stride"),
    (dict(batch=3, stride=9), "overlap"), (dict(steps=99), "steps"), (dict(products=5), "products"),
    (dict(m=C.c_void_p(0x10002)), "aligned"), (dict(work=None, rows=300), "workspace"), (dict(nbytes=1, rows=300), "workspace"),
    (dict(rows=1 << 17), "rows"), (dict(eps=-0.5), "eps"),
])
def test_muon_refuses(pkg, kw, word):
    lib = pkg.lib()
    assert _muon(lib, **kw) != 0
    assert word in lib.cfp_last_error().decode()


@pytest.mark.parametrize("kw", [
    dict(out=C.c_void_p(0x10004)), dict(ldo=65), dict(batch=2, so=64 * 65), dict(out=C.c_void_p(0x10000 + 64 * 64 * 4 - 4)),
    dict(ld=127, ldo=127, out=C.c_void_p(0x10000 + 64 * 4)), dict(ld=128, ldo=128, out=C.c_void_p(0x10000 + 63 * 4)),
    dict(ld=128, ldo=128, out=C.c_void_p(0x10000 + 65 * 4)),
])
def test_orthogonalize_refuses_an_output_across_the_input(pkg, kw):
    assert _ortho(pkg.lib(), **{**dict(rows=64, cols=64), **kw}) != 0
    assert b"overlap" in pkg.lib().cfp_last_error()


@pytest.mark.parametrize("kw", [
    dict(), dict(g=C.c_void_p(0x10000 + BIG)), dict(m=C.c_void_p(0x10000 + BIG)), dict(w=C.c_void_p(0x10000 + BIG)),
    dict(g=C.c_void_p(0x10000 + 64 * 64 * 4), m=C.c_void_p(0x10000 + 64 * 64 * 8 - 4)),
])
def test_muon_refuses_arrays_across_each_other(pkg, kw):
    assert _muon(pkg.lib(), **kw) != 0
    assert b"overlap" in pkg.lib().cfp_last_error()


def test_no_matrices_is_no_work(pkg):
    assert _ortho(pkg.lib(), batch=0, g=None, out=None, work=None, nbytes=0) == 0
    assert _muon(pkg.lib(), batch=0, w=None, g=None, m=None, work=None, nbytes=0) == 0


def test_workspace_sizes(pkg):
    ws = pkg.lib().cfp_orthogonalize_workspace
    assert ws(0, 64, 64, 1) == 0 and ws(1, 0, 64, 1) == 0 and ws(1, 64, 64, 2) == 0 and ws(1, 64, 1 << 17, 1) == 0
    assert ws(9, 64, 256, 3) == 0 and ws(1, 128, 128, 1) == 0     # one workgroup, no workspace
    assert ws(1, 128, 128, 3) > 0 and ws(1, 64, 300, 3) > 0 and ws(1, 128, 160, 1) > 0
    one, three = ws(1, 1000, 3000, 1), ws(1, 1000, 3000, 3)
    # three matrices of the gradient's size and two of the shorter side squared, at least
    assert one >= 2 * (3 * 1000 * 3000 + 2 * 1000 * 1000) and three > one
    assert ws(1, 3000, 1000, 3) == three and ws(4, 1000, 3000, 3) > 3 * three
    assert ws(1, 1 << 16, 1 << 16, 3) > 1 << 33     # sizes are not cut to 32 bits


def test_python_checks_before_the_library(pkg):
    import torch
    with pytest.raises(ValueError, match="g:"):
        pkg.policy.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="w:"):
        pkg.policy.muon_update(torch.zeros(4, 4), torch.zeros(4, 4), torch.zeros(4, 4), 0.1)


def test_optimizer_refusals(pkg):
    lib = pkg.lib()
    cfg = pkg._lib.MuonConfig()
    assert lib.cfp_muon_defaults(C.byref(cfg)) == 0 and cfg.steps == 5 and cfg.nesterov == 1
    assert lib.cfp_muon_defaults(None) != 0
    assert lib.cfp_train_set_optimizer(None, 1, None, None) != 0 and b"NULL" in lib.cfp_last_error()
    assert lib.cfp_train_muon(None, None) != 0 and lib.cfp_train_optimizer(None) == -1


@pytest.mark.parametrize("scale", [-1.0, -1e-30, float("nan")])
def test_muon_refuses_a_scale_below_zero(pkg, scale):
    """0 asks for the default; below it nothing is meant."""
    lib = pkg.lib()
    far = [C.c_void_p(0x10000 + k * BIG) for k in range(3)]
    assert lib.cfp_muon_update(*far, 64, 4096, 1, 64, 64, None, 0.1, 0.9, 1, 0.0, scale, 5, None, 1e-7, 0, P, BIG, None) != 0
    assert b"scale" in lib.cfp_last_error()


def test_build_refuses_products_that_spill_or_outgrow_their_budget():
    """k_ortho_mul and k_ortho_pair wait for counted copies."""
    import __graft_entry__ as entry
    build = entry._load_build_module()

    def remarks(name, vgprs=80, agprs=32, scratch=0, occupancy=2):
        return "\n".join(f"x.hip:1:1: remark: {l} [-Rpass-analysis=kernel-resource-usage]" for l in (
            f"Function Name: _ZN3cfp12_GLOBAL__N_1{len(name)}{name}ILi3ELi0ELi1EEEv", f"    VGPRs: {vgprs}", f"    AGPRs: {agprs}",
            f"    ScratchSize [bytes/lane]: {scratch}", f"    Occupancy [waves/SIMD]: {occupancy}"))

    for name in ("k_ortho_mul", "k_ortho_pair"):
        build.check_no_scratch(remarks(name))
        build.check_counted_wait_budget(remarks(name))
        with pytest.raises(RuntimeError, match=name):
            build.check_no_scratch(remarks(name, scratch=16))
        for kw in (dict(vgprs=200), dict(agprs=300), dict(occupancy=0), dict(occupancy=4)):
            with pytest.raises(RuntimeError, match=name):
                build.check_counted_wait_budget(remarks(name, **kw))
