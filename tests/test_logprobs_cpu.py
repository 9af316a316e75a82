"""Argument checks of cfp_token_logprobs / cfp_token_logprobs_grad: every refusal comes
before the first HIP call, so none of this needs a GPU."""
import ctypes as C

import pytest

P = C.c_void_p(0x10000)   # never dereferenced: each call below is refused on the host


def _forward(lib, dtype=0, ld=300, rows=2, vocab=300, mask=None, ldm=0, x=P, tok=P, lp=P, top=0, ids=None,
             tlp=None, work=None, nbytes=0):
    return lib.cfp_token_logprobs(x, dtype, ld, rows, vocab, tok, mask, ldm, lp, None, top, ids, tlp, None,
                                  work, nbytes, None)


def _grad(lib, dtype=0, ld=300, rows=2, vocab=300, x=P, stats=P, dx=C.c_void_p(0x900000), ldd=300, top=0,
          ids=None, g_top=None, mask=None, ldm=0):
    return lib.cfp_token_logprobs_grad(x, dtype, ld, rows, vocab, P, mask, ldm, stats, None, None, top, ids,
                                       g_top, dx, ldd, None)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 30) + 1, ld=1 << 31), "vocab"), (dict(top=33, ids=P, tlp=P), "top"), (dict(top=-1), "top"),
    (dict(x=None), "NULL"), (dict(tok=None), "NULL"), (dict(lp=None), "NULL"), (dict(ld=299), "stride"),
    (dict(mask=P, ldm=299), "mask"), (dict(top=4, ids=P), "alternatives"), (dict(top=4, tlp=P), "alternatives"),
    (dict(x=C.c_void_p(0x10002)), "aligned"), (dict(dtype=1, x=C.c_void_p(0x10001)), "aligned"),
    (dict(rows=1, vocab=131072, ld=131072), "workspace"),
    (dict(rows=1, vocab=131072, ld=131072, work=P, nbytes=16), "workspace"),
    (dict(rows=1, vocab=131072, ld=131072, work=C.c_void_p(0x10008), nbytes=1 << 20), "workspace"),
    (dict(rows=(1 << 31) - 1, vocab=8193, ld=8193), "more than one launch"),
])
def test_forward_refuses(pkg, kw, word):
    lib = pkg.lib()
    assert _forward(lib, **kw) != 0
    assert word in lib.cfp_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"), (dict(stats=None), "NULL"), (dict(dx=None), "NULL"), (dict(x=None), "NULL"),
    (dict(ldd=299), "stride"), (dict(ld=299), "stride"), (dict(top=2, ids=P), "gradients"),
    (dict(top=40, ids=P, g_top=P), "top"), (dict(dx=C.c_void_p(0x900001)), "aligned"),
    (dict(dx=C.c_void_p(0x10004)), "overlap"), (dict(dx=P, ldd=301), "overlap"),
    (dict(dx=C.c_void_p(0x10000 - 4), ldd=300), "overlap"), (dict(mask=P, ldm=1), "mask"),
])
def test_gradient_refuses(pkg, kw, word):
    lib = pkg.lib()
    assert _grad(lib, **kw) != 0
    assert word in lib.cfp_last_error().decode()


def test_no_rows_is_no_work(pkg):
    lib = pkg.lib()
    assert _forward(lib, rows=0, x=None, tok=None, lp=None) == 0
    assert lib.cfp_token_logprobs_grad(None, 1, 0, 0, 5, None, None, 0, None, None, None, 0, None, None, None, 0,
                                       None) == 0


def test_workspace_sizes(pkg):
    ws = pkg.lib().cfp_token_logprobs_workspace
    assert ws(4096, 43, 32) == 0 and ws(4096, 131072, 5) == 0 and ws(0, 131072, 5) == 0
    assert ws(1, 131072, 0) >= 2 * 16 and ws(1, 131072, 32) > ws(1, 131072, 0)
    assert ws(1, 0, 0) == 0 and ws(1, 100, 33) == 0


def test_python_checks_before_the_library(pkg):
    import torch
    pol = pkg.policy
    x, t = torch.zeros(4, 43), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="logits"):
        pol.token_logprobs(x, t)
    with pytest.raises(ValueError, match="logits"):
        pol.token_logprobs_backward(x, t, torch.zeros(4, 3))
