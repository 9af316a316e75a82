"""cfp_token_logprobs / cfp_token_logprobs_grad against the definition in 64 bits.

Tolerances, with u = 2^-24 (one fp32 rounding), D the distance from the row's maximum that an
entry of any weight has (entries more than 100 below it weigh under e^-100), k the entries one
lane adds up: every exponent y = (x - m) log2 e carries two roundings (2 u |y|), its
exponential one unit in the last place (2 u), a lane's sum k u, the tree over lanes and
wavefronts at most 12 u, each raise of the maximum another pair of roundings (fewer than k of
them).  So ln s is off by at most u (4 D + 2 k + 32) and so is ln p with the two subtractions
(u |x - m| + u |ln s|) inside the same bound; the entropy weighs each of those errors by
1 + H at most (E[m - x] <= H)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _torch():
    import torch
    return torch


DT = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def make(cuda, dtype, rows, vocab, ld=None, seed=0, spread=2.5, offset=0):
    """[rows][vocab] logits as a view of rows `ld` wide that begins `offset` elements in."""
    torch = _torch()
    ld = ld or vocab
    g = torch.Generator(device="cpu").manual_seed(seed)
    store = torch.full((offset + rows * ld,), 7.0, dtype=getattr(torch, DT[dtype]))
    x = store[offset:].view(rows, ld)[:, :vocab]
    x.copy_(torch.randn(rows, vocab, generator=g) * spread)
    dev = store.to(cuda)
    tok = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    return dev[offset:].view(rows, ld)[:, :vocab], tok.to(cuda)


def reference(x, tok, mask, top):
    """The definition in float64 on the CPU: (lp, entropy, ids, top lp, log p with -inf where
    not allowed, distance D of each row)."""
    torch = _torch()
    x = x.double().cpu()
    rows, vocab = x.shape
    ok = torch.ones(rows, vocab, dtype=torch.bool) if mask is None else (mask.cpu() != 0).expand(rows, vocab)
    ok = ok & (x != -torch.inf)
    z = torch.where(ok, x, -torch.inf)
    some = ok.any(1)
    bad = (torch.where(ok, x, 0.0).isnan() | (z == torch.inf)).any(1)
    m = torch.where(some, z.amax(1), 0.0)[:, None]
    d = z - m
    s = torch.where(ok, d.exp(), 0.0).sum(1, keepdim=True)
    logp = torch.where(ok, d - s.log(), -torch.inf)
    p = torch.where(ok, logp.exp(), 0.0)
    ent = -(p * torch.where(ok, logp, 0.0)).sum(1)
    t = tok.cpu().long()
    lp = logp.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0]
    lp = torch.where(bad | (t >= vocab), torch.nan, lp)
    lp = torch.where(t < 0, 0.0, lp)
    ent = torch.where(bad, torch.nan, ent)
    order = torch.sort(torch.where(ok & ~bad[:, None], x, -torch.inf), dim=1, descending=True, stable=True)[1][:, :top]
    there = ok.gather(1, order) & ~bad[:, None]
    tlp = torch.where(there, logp.gather(1, order), -torch.inf)
    tlp = torch.where(bad[:, None], torch.nan, tlp)
    ids = torch.where(there, order, -1)
    if top > vocab:
        ids = torch.nn.functional.pad(ids, (0, top - vocab), value=-1)
        tlp = torch.cat([tlp, torch.where(bad[:, None], torch.nan, -torch.inf).expand(rows, top - vocab)], 1)
    reach = torch.where(ok & ~bad[:, None], -d, 0.0).clamp(0, 100).amax(1)
    return lp, ent, ids, tlp, logp, reach


def lane_entries(vocab):
    """k: entries one lane adds up at most (one wavefront a row up to 8192, else 256 lanes of a
    workgroup; partial tiles count whole)."""
    return 4 if vocab <= 256 else (vocab if vocab <= 8192 else vocab // 4) // 64 + 64


def close(got, want, tol, what):
    got, want = got.double().cpu().numpy(), want.numpy()
    tol = np.broadcast_to(np.asarray(tol), want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    keep = ~fin & ~np.isnan(want)
    assert np.array_equal(got[keep], want[keep]), what
    off = np.abs(got[fin] - want[fin]) - tol[fin]
    assert off.size == 0 or off.max() <= 0, f"{what}: {off.max()} over the tolerance"


def check_forward(pkg, x, tok, mask=None, top=0):
    got = pkg.policy.token_logprobs(x, tok, mask=mask, top=top, stats=True)
    lp, ent, ids, tlp, logp, reach = reference(x, tok, mask, top)
    k = lane_entries(x.shape[1])
    t = tok.cpu().long().clamp(0, x.shape[1] - 1)
    far = np.nan_to_num(np.abs(lp.numpy()), posinf=0.0)
    tol = U * (4 * reach.numpy() + 2 * k + 32 + 4 * far)
    close(got.logprobs, lp, tol, "logprobs")
    close(got.entropy, ent, U * (4 * reach.numpy() + 2 * k + 32) * (1 + np.nan_to_num(ent.numpy())), "entropy")
    if top:
        assert np.array_equal(got.top_ids.cpu().numpy(), ids.numpy().astype(np.int32)), "top ids"
        close(got.top_logprobs, tlp,
              (U * (4 * reach.numpy() + 2 * k + 32))[:, None] + 4 * U * np.nan_to_num(np.abs(tlp.numpy()), posinf=0.0),
              "top logprobs")
    else:
        assert got.top_ids is None and got.top_logprobs is None
    return got, t


SHAPES = [(1, 1), (3, 2), (5, 16), (7, 17), (33, 43), (64, 64), (9, 65), (2, 255), (11, 256), (6, 257), (1, 511),
          (5, 1000), (4096, 300), (4100, 2049), (2, 4096), (3, 8192), (1, 8200), (2, 50021), (1, 131072),
          (16384, 1), (16400, 8), (16390, 31), (16500, 43), (20001, 64)]      # one thread a row


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward_against_64_bits(pkg, cuda, dtype, rows, vocab):
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + (3 if rows > 1 else 0), seed=rows + vocab)
    check_forward(pkg, x, tok, top=min(32, vocab + 2))
    check_forward(pkg, x, tok)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,top", [(40, 43, 5), (37, 200, 32), (29, 1021, 20), (4099, 777, 3), (31, 9001, 8),
                                            (2, 70001, 20), (16390, 43, 0), (16390, 17, 2)])
@pytest.mark.parametrize("shared", [False, True])
def test_masks_empty_rows_and_padding(pkg, cuda, dtype, rows, vocab, top, shared):
    """Masks per row and one for all rows, NaN and infinities behind them, rows that allow
    nothing or one entry, padding tokens, tokens that are masked, tokens past the row."""
    torch = _torch()
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + 1, seed=5, offset=1)
    g = torch.Generator(device="cpu").manual_seed(9)
    mask = (torch.rand(vocab if shared else rows * vocab, generator=g) < 0.5).to(torch.uint8)
    mask = (mask if shared else mask.view(rows, vocab)).to(cuda)
    full = mask.expand(rows, vocab)
    hidden = x.clone()
    junk = torch.tensor([float("nan"), float("inf"), -float("inf")], device=cuda).to(x.dtype)
    x[:] = torch.where(full == 0, junk[torch.arange(vocab, device=cuda) % 3], hidden)
    if not shared:
        mask[1::5] = 0
        mask[0] = 0
        mask[0, vocab // 2] = 1
        x[0, vocab // 2] = 1.5
        x[1::5] = float("nan")
        # entries that the mask now hides or shows hold finite values only where allowed
    tok[::7] = -1
    tok[rows - 1] = vocab
    got, _ = check_forward(pkg, x, tok, mask=mask, top=top)
    if not shared:
        assert got.entropy[1].item() == 0 and got.entropy[0].item() == 0
        assert not top or got.top_ids[1].eq(-1).all()
    # a bool mask is the same mask
    other = pkg.policy.token_logprobs(x, tok, mask=mask.bool(), top=top)
    assert torch.equal(other.entropy.nan_to_num(7.0), got.entropy.nan_to_num(7.0))


@pytest.mark.parametrize("vocab", [43, 200, 3000, 20000])
def test_border_values(pkg, cuda, vocab):
    torch = _torch()
    low = torch.finfo(torch.float32).min
    x = torch.zeros(9, vocab, device=cuda)
    x[0] = low                                  # every entry the type's lowest: uniform
    x[1] = low; x[1, vocab - 1] = 3.0           # one entry stands out
    x[2] = -float("inf")                        # nothing allowed
    x[3] = -float("inf"); x[3, 1] = -4.0        # one entry
    x[4, 2] = float("nan")
    x[5, 2] = float("inf")
    x[6] = 1.0e30; x[6, 0] = -1.0e30            # wide range
    x[7] = 3.0e4 + torch.arange(vocab, device=cuda) % 7   # large offset: bits of ln s must survive
    tok = torch.full((9,), 1, dtype=torch.int32, device=cuda)
    tok[1] = vocab - 1
    tok[8] = 0
    check_forward(pkg, x, tok, top=5)
    for r in range(9):                          # alone: the split kernels where rows are few
        check_forward(pkg, x[r:r + 1], tok[r:r + 1], top=5)


@pytest.mark.parametrize("dtype,vocab", [("bf16", 40), ("bf16", 250), ("bf16", 5000), ("f16", 33000), ("f32", 9000)])
def test_ties_go_to_the_lowest_index(pkg, cuda, dtype, vocab):
    torch = _torch()
    x, tok = make(cuda, dtype, 4, vocab, seed=3)
    x[0] = 0.0
    x[0, ::2] = -0.0                            # equal zeros
    x[1] = torch.arange(vocab, device=cuda).remainder(3).to(x.dtype)
    x[2] = -torch.arange(vocab, device=cuda).to(x.dtype)          # sorted, rounded: runs of equals
    x[3] = torch.arange(vocab, device=cuda).to(x.dtype)
    got, _ = check_forward(pkg, x, tok, top=32)
    assert got.top_ids[0].tolist() == list(range(32))


def grad_reference(x, tok, mask, g_lp, g_ent, ids, g_top):
    """Gradient in float64 and the tolerance of each entry before its last rounding."""
    torch = _torch()
    lp, ent, _, _, logp, reach = reference(x, tok, mask, 0)
    rows, vocab = x.shape
    ok = logp > -torch.inf
    p = torch.where(ok, logp.exp(), 0.0)
    l = torch.where(ok, logp, 0.0)
    t = tok.cpu().long()
    live = (t >= 0) & ok.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0]
    g = torch.where(live, g_lp.double().cpu(), 0.0) if g_lp is not None else torch.zeros(rows, dtype=torch.float64)
    hot = torch.zeros(rows, vocab, dtype=torch.float64)
    hot.scatter_add_(1, t.clamp(0, vocab - 1)[:, None], g[:, None])
    w = g.clone()
    size = g.abs()
    if g_top is not None:
        i = ids.cpu().long()
        a = torch.where((i >= 0) & ok.gather(1, i.clamp(0, vocab - 1)), g_top.double().cpu(), 0.0)
        hot.scatter_add_(1, i.clamp(0, vocab - 1), a)
        w = w + a.sum(1)
        size = size + a.abs().sum(1)
    h = torch.zeros(rows, dtype=torch.float64) if g_ent is None else g_ent.double().cpu()
    want = torch.where(ok, hot - p * (w[:, None] + h[:, None] * (l + ent[:, None])), 0.0)
    e_l = U * (4 * reach + 2 * lane_entries(vocab) + 32)[:, None] + 4 * U * l.abs()   # of ln p
    e_h = (U * (4 * reach + 2 * lane_entries(vocab) + 32) * (1 + ent))[:, None]
    inner = size[:, None] + h.abs()[:, None] * (l.abs() + ent[:, None])
    tol = p * (inner * (e_l + 40 * U) + h.abs()[:, None] * (e_l + e_h)) + 8 * U * (hot.abs() + size[:, None] * (hot != 0))
    return want, tol


def check_grad(pkg, x, tok, mask=None, top=0, lp=True, ent=True, seed=1, out=None):
    torch = _torch()
    rows = x.shape[0]
    g = torch.Generator(device="cpu").manual_seed(seed)
    g_lp = torch.randn(rows, generator=g).to(x.device) if lp else None
    g_ent = torch.randn(rows, generator=g).to(x.device) if ent else None
    g_top = torch.randn(rows, top, generator=g).to(x.device) if top else None
    got = pkg.policy.token_logprobs(x, tok, mask=mask, top=top, stats=True)
    want, tol = grad_reference(x, tok, mask, g_lp, g_ent, got.top_ids, g_top)
    dx = pkg.policy.token_logprobs_backward(x, tok, got.stats, g_logprobs=g_lp, g_entropy=g_ent, mask=mask,
                                            top_ids=got.top_ids, g_top=g_top, out=out)
    fi = torch.finfo(x.dtype)
    step = want.abs() * fi.eps / 2 + fi.tiny * fi.eps / 2   # rounding once to the type, denormals included
    # a value next to a rounding border may fall to the other side: a whole step there
    tol = tol.numpy() * (1 + fi.eps) + step.numpy()
    close(dx, want, tol, "gradient")
    return got, dx, (g_lp, g_ent, g_top)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (5, 2), (33, 43), (7, 64), (6, 65), (9, 256), (5, 257), (3, 4099),
                                        (2, 8192), (1, 16385), (2, 50021), (1, 131072), (16384, 5), (16390, 9), (16500, 43),
                                        (20001, 64)])
def test_gradient_against_the_formula(pkg, cuda, dtype, rows, vocab):
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + (5 if rows > 1 else 0), seed=vocab)
    check_grad(pkg, x, tok)
    check_grad(pkg, x, tok, top=min(32, vocab + 1), seed=2)
    check_grad(pkg, x, tok, lp=False, seed=3)
    check_grad(pkg, x, tok, ent=False, seed=4)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(37, 43), (21, 130), (11, 3001), (3, 40001), (16390, 43)])
def test_gradient_under_masks(pkg, cuda, dtype, rows, vocab):
    torch = _torch()
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + 1, seed=4, offset=1)
    g = torch.Generator(device="cpu").manual_seed(2)
    mask = (torch.rand(rows, vocab, generator=g) < 0.6).to(torch.uint8).to(cuda)
    x[:] = torch.where(mask == 0, torch.full_like(x, float("nan")), x)
    mask[1::4] = 0
    tok[2::5] = -1
    check_grad(pkg, x, tok, mask=mask, seed=2)
    got, dx, _ = check_grad(pkg, x, tok, mask=mask, top=8)
    assert dx[1].eq(0).all() and dx[mask == 0].eq(0).all()


@pytest.mark.parametrize("rows,vocab,top", [(50, 43, 5), (5, 300, 5), (3, 30001, 5), (16400, 43, 0)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_in_place_of_the_logits(pkg, cuda, dtype, rows, vocab, top):
    torch = _torch()
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + 2, seed=6)
    got, dx, gs = check_grad(pkg, x, tok, top=top)
    again = pkg.policy.token_logprobs_backward(x, tok, got.stats, g_logprobs=gs[0], g_entropy=gs[1],
                                               top_ids=got.top_ids, g_top=gs[2], out=x)
    assert again is x and torch.equal(x, dx)


def test_the_same_alternative_twice(pkg, cuda):
    torch = _torch()
    for vocab in (50, 5000):
        x, tok = make(cuda, "f32", 3, vocab, seed=8)
        got = pkg.policy.token_logprobs(x, tok, stats=True)
        ids = torch.stack([tok, tok, torch.full_like(tok, 7), torch.full_like(tok, 7), torch.full_like(tok, -1)], 1)
        g_top = torch.arange(1, 16, device=cuda).float().view(3, 5)
        g_lp = torch.ones(3, device=cuda)
        want, tol = grad_reference(x, tok, None, g_lp, None, ids, g_top)
        dx = pkg.policy.token_logprobs_backward(x, tok, got.stats, g_logprobs=g_lp, top_ids=ids.contiguous(), g_top=g_top)
        close(dx, want, tol.numpy() + U * want.abs().numpy() + 64 * U, "gradient")


def test_an_index_past_the_row_is_not_quiet(pkg, cuda):
    torch = _torch()
    for vocab in (43, 700):
        x, tok = make(cuda, "f32", 4, vocab, seed=8)
        tok[2] = vocab
        got = pkg.policy.token_logprobs(x, tok, stats=True)
        dx = pkg.policy.token_logprobs_backward(x, tok, got.stats, g_logprobs=torch.ones(4, device=cuda))
        assert got.logprobs[2].isnan() and dx[2].isnan().all() and not dx[[0, 1, 3]].isnan().any()


def test_gradient_against_differences(pkg, cuda):
    """(f(x + h v) - f(x - h v)) / 2h of the kernel's own values along a direction v of +-1.
    h = 2^-5: the cut-off is h^2/6 of a third derivative, at most 2 |g| for the log-probability
    (third central moment of values in [-1, 1], twice over) and 2 |g_H| (ln vocab + D + 8) for
    the entropy; the values' own errors (test_forward's bound, twice) come divided by 2 h."""
    torch = _torch()
    rows, vocab, h = 64, 43, 2.0 ** -5
    x, tok = make(cuda, "f32", rows, vocab, seed=12, spread=1.5)
    got, dx, (g_lp, g_ent, _) = check_grad(pkg, x, tok)
    gen = torch.Generator(device="cpu").manual_seed(3)
    v = (torch.randint(0, 2, (rows, vocab), generator=gen) * 2 - 1).float().to(cuda)

    def f(y):
        r = pkg.policy.token_logprobs(y, tok)
        return (g_lp.double() * r.logprobs.double() + g_ent.double() * r.entropy.double())

    # x +- h v is rounded: the step that was really taken
    up, dn = x + h * v, x - h * v
    diff = (f(up) - f(dn)) / (2 * h)
    along = (dx.double() * v.double()).sum(1)
    reach = 12.0
    cut = h * h / 6 * (2 * g_lp.abs() + 2 * g_ent.abs() * (np.log(vocab) + reach + 8)).double()
    noise = (g_lp.abs() + g_ent.abs() * 5).double() * U * (4 * reach + 40 + 48) / h + 2 * U * 8 * vocab * dx.abs().amax(1).double() / h
    assert ((diff - along).abs() <= cut + noise).all()


@pytest.mark.parametrize("vocab", [100, 3000])
def test_offsets_past_32_bits(pkg, cuda, vocab):
    """Rows 2^30 + 9 elements apart: the third starts past 2^31 elements, 4 GiB in."""
    torch = _torch()
    ld = (1 << 30) + 9
    store = torch.empty(2 * ld + vocab, dtype=torch.bfloat16, device=cuda)
    x = torch.as_strided(store, (3, vocab), (ld, 1))
    small, tok = make(cuda, "bf16", 3, vocab, seed=2)
    x.copy_(small)
    a = pkg.policy.token_logprobs(x, tok, top=7, stats=True)
    b = pkg.policy.token_logprobs(small, tok, top=7, stats=True)
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    g = torch.ones(3, device=cuda)
    want = pkg.policy.token_logprobs_backward(small, tok, b.stats, g_logprobs=g, g_entropy=g)
    pkg.policy.token_logprobs_backward(x, tok, a.stats, g_logprobs=g, g_entropy=g, out=x)
    assert torch.equal(x, want)


def test_rows_behind_the_last_are_left_alone(pkg, cuda):
    """Output arrays with room for more rows, and rows wider than the logits."""
    torch = _torch()
    lib = pkg.lib()
    for rows, vocab, top in ((19, 43, 3), (5, 120, 3), (5, 3000, 3), (1, 20000, 3), (16387, 43, 0)):
        x, tok = make(cuda, "f32", rows, vocab, ld=vocab + 4, seed=rows)
        wide = torch.full((rows + 2, vocab + 4), 9.0, device=cuda)
        f = [torch.full((rows + 2,), 5.0, device=cuda) for _ in range(2)]
        st = torch.full((rows + 2, 3), 5.0, device=cuda)
        ids = torch.full((rows + 2, max(top, 1)), 77, dtype=torch.int32, device=cuda)
        tlp = torch.full((rows + 2, max(top, 1)), 5.0, device=cuda)
        n = lib.cfp_token_logprobs_workspace(rows, vocab, top)
        work = torch.full((n + 16,), 3, dtype=torch.uint8, device=cuda)
        stream = torch.cuda.current_stream().cuda_stream
        assert lib.cfp_token_logprobs(x.data_ptr(), 0, vocab + 4, rows, vocab, tok.data_ptr(), None, 0, f[0].data_ptr(),
                                      f[1].data_ptr(), top, ids.data_ptr(), tlp.data_ptr(), st.data_ptr(),
                                      work.data_ptr(), n, stream) == 0
        assert lib.cfp_token_logprobs_grad(x.data_ptr(), 0, vocab + 4, rows, vocab, tok.data_ptr(), None, 0, st.data_ptr(),
                                           f[0].data_ptr(), None, 0, None, None, wide.data_ptr(), vocab + 4, stream) == 0
        torch.cuda.synchronize()
        for t in (*f, st, tlp)[:4 if top else 3]:
            assert t[rows:].eq(5.0).all() and not t[:rows].eq(5.0).any()
        assert ids[rows:].eq(77).all() and work[n:].eq(3).all()
        assert wide[rows:].eq(9.0).all() and wide[:, vocab:].eq(9.0).all() and not wide[:rows, :vocab].eq(9.0).any()


def test_same_call_same_bits_on_any_stream_and_from_a_graph(pkg, cuda):
    torch = _torch()
    pol = pkg.policy
    for rows, vocab, dtype, top in ((300, 43, "f32", 6), (4096, 500, "bf16", 6), (3, 60000, "bf16", 6), (16500, 43, "f32", 0)):
        x, tok = make(cuda, dtype, rows, vocab, seed=1)
        g = torch.randn(rows, device=cuda)

        def both():
            r = pol.token_logprobs(x, tok, top=top, stats=True)
            d = pol.token_logprobs_backward(x, tok, r.stats, g_logprobs=g, g_entropy=g, top_ids=r.top_ids,
                                            g_top=r.top_logprobs)
            return (*(t for t in r if t is not None), d)

        want = [t.clone() for t in both()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for t, w in zip(both(), want):
                assert torch.equal(t, w)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both()
        keep = x.clone()
        for rep in range(3):
            x.copy_(keep if rep != 1 else keep * 0.5)
            eager = [t.clone() for t in both()]
            for t in outs:
                t.fill_(3)
            graph.replay()
            torch.cuda.synchronize()
            for t, w in zip(outs, eager):
                assert torch.equal(t, w)
        x.copy_(keep)


def test_scores_of_the_policy_own_actions(pkg, cuda):
    """forward -> heads -> sample, then the sampled actions scored from the same head rows: the
    log-probabilities are cfp_value_sample's."""
    torch = _torch()
    n = 256
    pol = pkg.Policy(n, layers=2, seed=4)
    rec = pkg.policy.synth_records(n, 11, 0)
    av = pol.forward(rec, torch.zeros(n, device=cuda), torch.zeros((2, n, 256), device=cuda))
    act, lp, _ = pkg.policy.value_sample(av, 17)
    got, _ = check_forward(pkg, av[:, :43], act, top=4)
    assert (got.logprobs - lp).abs().max().item() <= 2 * U * (4 * 20 + 2 * 43 + 64)
    pol.close()


def test_refusals_with_device_tensors(pkg, cuda):
    torch = _torch()
    pol = pkg.policy
    x, tok = make(cuda, "f32", 4, 43, seed=1)
    st = torch.zeros(4, 3, device=cuda)
    for bad in (lambda: pol.token_logprobs(x, tok.long()), lambda: pol.token_logprobs(x, tok[:3]),
                lambda: pol.token_logprobs(x.double(), tok), lambda: pol.token_logprobs(x[0], tok),
                lambda: pol.token_logprobs(x.t(), tok), lambda: pol.token_logprobs(x, tok.cpu()),
                lambda: pol.token_logprobs(x, None),
                lambda: pol.token_logprobs(x, tok, mask=torch.ones(4, 42, dtype=torch.uint8, device=cuda)),
                lambda: pol.token_logprobs(x, tok, mask=torch.ones(4, 43, device=cuda)),
                lambda: pol.token_logprobs_backward(x, tok, None),
                lambda: pol.token_logprobs_backward(x, tok, st, g_top=torch.zeros(4, 2, device=cuda)),
                lambda: pol.token_logprobs_backward(x, tok, st, g_logprobs=torch.zeros(3, device=cuda)),
                lambda: pol.token_logprobs_backward(x, tok, st, out=torch.zeros(4, 43, device=cuda, dtype=torch.float16))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg._lib.CfpError, match="top"):
        pol.token_logprobs(x, tok, top=33)
    with pytest.raises(pkg._lib.CfpError, match="stride"):
        pol.token_logprobs(x[:1].expand(4, 43), tok)
    with pytest.raises(pkg._lib.CfpError, match="overlap"):
        wide = torch.zeros(4, 90, device=cuda)
        pol.token_logprobs_backward(wide[:, :43], tok, st, out=wide[:, 20:63])
    assert pol.token_logprobs(x[:0], tok[:0]).logprobs.numel() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 131072), (2, 50021), (7, 2100), (300, 40001), (3000, 17000)])
def test_in_place_with_named_entries_that_are_not_allowed(pkg, cuda, dtype, rows, vocab):
    """Tokens and alternatives at -inf, spread over the whole row, with gradients of their own: they
    pass nothing on, whichever part of the row is replaced first.  In 16 bits some gradients that
    replace a logit overflow to -inf.  Bit for bit as into another array."""
    torch = _torch()
    pol = pkg.policy
    x, tok = make(cuda, dtype, rows, vocab, seed=21)
    at = torch.arange(rows, device=cuda)
    tok[:] = ((at * 7919 + vocab // 3) % vocab).int()
    named = torch.stack([(at * 131 + k * (vocab // 9) + 5) % vocab for k in range(9)], 1).int()
    off_ = at % 4 != 3                        # three rows of four: the token is not allowed
    x[at[off_], tok[off_].long()] = -torch.inf
    x.scatter_(1, named[:, ::2].long(), -torch.inf)
    mask = None if dtype == "f32" else torch.ones(vocab, dtype=torch.uint8, device=cuda)
    got = pol.token_logprobs(x, tok, mask=mask, stats=True)
    g = torch.Generator(device="cpu").manual_seed(5)
    g_lp, g_ent = (torch.randn(rows, generator=g).to(cuda) for _ in range(2))
    g_lp *= 1e9 if dtype == "f16" else 1.0
    g_top = torch.randn(rows, 9, generator=g).to(cuda)
    for ids, gt in ((None, None), (named.contiguous(), g_top)):
        kw = dict(g_logprobs=g_lp, g_entropy=g_ent, mask=mask, top_ids=ids, g_top=gt)
        want = pol.token_logprobs_backward(x, tok, got.stats, **kw)
        ref, tol = grad_reference(x[:8], tok[:8], mask, g_lp[:8], g_ent[:8], None if ids is None else ids[:8],
                                  None if gt is None else gt[:8])
        if dtype == "f32":
            close(want[:8], ref, tol.numpy() + U * ref.abs().numpy() + 2.0 ** -149, "gradient")
        for _ in range(3):
            y = x.clone()
            pol.token_logprobs_backward(y, tok, got.stats, out=y, **kw)
            assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(16384, 8), (16384, 42), (16500, 42), (16512, 64), (16391, 10)])
@pytest.mark.parametrize("in_place", [False, True])
def test_one_column_behind_even_rows_is_left_alone(pkg, cuda, dtype, rows, vocab, in_place):
    """Rows vocab + 1 apart, as a head's logits with a value behind them: the gradient leaves that
    column and what follows the last logit as they were."""
    torch = _torch()
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + 1, seed=vocab)
    got = pkg.policy.token_logprobs(x, tok, stats=True)
    g = torch.randn(rows, generator=torch.Generator().manual_seed(2)).to(cuda)
    want = pkg.policy.token_logprobs_backward(x.contiguous(), tok, got.stats, g_logprobs=g, g_entropy=g)
    store = torch.full((rows * (vocab + 1) + 64,), 9.0, dtype=x.dtype, device=cuda)
    out = store[:rows * (vocab + 1)].view(rows, vocab + 1)[:, :vocab]
    assert out.data_ptr() % 16 == 0
    if in_place:
        out.copy_(x)
    dx = pkg.policy.token_logprobs_backward(out if in_place else x, tok, got.stats, g_logprobs=g, g_entropy=g, out=out)
    assert torch.equal(dx, want)
    assert store[:rows * (vocab + 1)].view(rows, vocab + 1)[:, vocab].eq(9).all() and store[rows * (vocab + 1) - 1:].eq(9).all()


@pytest.mark.parametrize("rows,vocab", [((1 << 30) + 300, 8), ((1 << 31) - 1, 2)])
def test_row_counts_past_30_bits(pkg, cuda, rows, vocab):
    """More rows than a 32-bit loop over them can step past, by one thread a row and by lanes: rows at
    the start, around 2^30 and at the end as in a call of their own, bit for bit."""
    torch = _torch()
    pol = pkg.policy
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GiB of free GPU memory")
    part = 16384 + 77
    cuts = [slice(a, a + part) for a in (0, (1 << 30) - part // 2, rows - part)]
    cuts = [c for c in cuts if c.stop <= rows]
    x = torch.zeros((rows, vocab), dtype=torch.float16, device=cuda)
    tok = torch.zeros(rows, dtype=torch.int32, device=cuda)
    g = torch.zeros(rows, dtype=torch.float32, device=cuda)
    for c in cuts:
        x[c] = torch.randn(part, vocab, device=cuda).half()
        tok[c] = torch.randint(-1, vocab, (part,), dtype=torch.int32, device=cuda)
        g[c] = torch.randn(part, device=cuda)
    got = pol.token_logprobs(x, tok, stats=True)
    dx = pol.token_logprobs_backward(x, tok, got.stats, g_logprobs=g, g_entropy=g)
    for c in cuts:
        want = pol.token_logprobs(x[c].clone(), tok[c].clone(), stats=True)
        for a, b in ((got.logprobs, want.logprobs), (got.entropy, want.entropy), (got.stats, want.stats)):
            assert torch.equal(a[c], b)
        assert torch.equal(dx[c], pol.token_logprobs_backward(x[c].clone(), tok[c].clone(), want.stats, g_logprobs=g[c].clone(),
                                                              g_entropy=g[c].clone()))
    middle = slice(rows // 4, rows // 4 + 1000)      # equal logits, token 0
    assert (got.logprobs[middle] + np.log(vocab)).abs().max().item() <= 8 * U
    del x, tok, g, got, dx
    torch.cuda.empty_cache()


def test_what_can_be_scored_can_be_differentiated(pkg, cuda):
    """More rows too long for registers than one launch has workgroups."""
    torch = _torch()
    pol = pkg.policy
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GiB of free GPU memory")
    rows, vocab, part = (1 << 24) + 4000, 1025, 5000
    cuts = [slice(0, part), slice(rows - part, rows)]
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=cuda)
    tok = torch.zeros(rows, dtype=torch.int32, device=cuda)
    g = torch.ones(rows, device=cuda)
    for c in cuts:
        x[c] = torch.randn(part, vocab, device=cuda).bfloat16()
        tok[c] = torch.randint(-1, vocab, (part,), dtype=torch.int32, device=cuda)
        g[c] = torch.randn(part, device=cuda)
    keep = [x[c].clone() for c in cuts]
    got = pol.token_logprobs(x, tok, stats=True)
    dx = pol.token_logprobs_backward(x, tok, got.stats, g_logprobs=g, g_entropy=g)
    pol.token_logprobs_backward(x, tok, got.stats, g_logprobs=g, g_entropy=g, out=x)
    fi = torch.finfo(torch.bfloat16)
    for c, k in zip(cuts, keep):
        assert torch.equal(dx[c], x[c])
        want, tol = grad_reference(k, tok[c], None, g[c], g[c], None, None)
        close(dx[c], want, tol.numpy() * (1 + fi.eps) + want.abs().numpy() * fi.eps / 2 + fi.tiny * fi.eps / 2, "gradient")
    middle = dx[rows // 2]                      # equal logits, token 0: 1 - 1/1025, rounded to 1
    assert middle[0].item() == 1.0 and (middle[1:].float() + 1 / vocab).abs().max().item() <= 2.0 ** -8 / vocab
    del x
    del dx, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(40, 43), (5, 2500), (2, 30001), (16400, 40)])
def test_logits_and_gradient_as_columns_of_one_array(pkg, cuda, dtype, rows, vocab):
    """Side by side in rows of one array, and in every second row of it: no entry is shared."""
    torch = _torch()
    pol = pkg.policy
    x, tok = make(cuda, dtype, rows, vocab, seed=31)
    got = pol.token_logprobs(x, tok, stats=True)
    g = torch.randn(rows, generator=torch.Generator().manual_seed(4)).to(cuda)
    want = pol.token_logprobs_backward(x, tok, got.stats, g_logprobs=g, g_entropy=g)
    store = torch.full((rows, 4 * vocab), 9.0, dtype=x.dtype, device=cuda)
    for a, b in ((store[:, :vocab], store[:, vocab:2 * vocab]), (store[:, 2 * vocab:3 * vocab], store[:, :vocab]),
                 (store.view(2 * rows, 2 * vocab)[:rows, :vocab], store[:, vocab:2 * vocab])):
        store.fill_(9.0)
        a.copy_(x)
        assert pol.token_logprobs_backward(a, tok, got.stats, g_logprobs=g, g_entropy=g, out=b) is b
        assert torch.equal(b, want) and torch.equal(a, x)
        a.fill_(9.0); b.fill_(9.0)
        assert store.eq(9).all()
    for b in (store[:, vocab - 1:2 * vocab - 1], store.view(2 * rows, 2 * vocab)[:rows, 1:vocab + 1]):
        with pytest.raises(pkg._lib.CfpError, match="overlap"):
            pol.token_logprobs_backward(store[:, :vocab], tok, got.stats, g_logprobs=g, out=b)


@pytest.mark.parametrize("dtype,rows,vocab", [("bf16", 513, 1 << 22), ("f16", 1, 1 << 30), ("f32", 700, 1000003)])
def test_long_rows_keep_their_sums(pkg, cuda, dtype, rows, vocab):
    """One entry at 0 and all others at -0.65625, whose exponentials round the same way at every step
    of a long running sum (16 384 of them in a row: 2.3e-4).  A lane adds up 512 and part of a tile."""
    torch = _torch()
    torch.cuda.empty_cache()
    x = torch.full((rows, vocab), -0.65625, dtype=getattr(torch, DT[dtype]), device=cuda)
    tok = ((torch.arange(rows, device=cuda) * 7919) % vocab).int()
    x[torch.arange(rows, device=cuda), tok.long()] = 0.0
    got = pkg.policy.token_logprobs(x, tok, top=1)
    rest = (vocab - 1) * np.exp(-0.65625)
    ls = np.log1p(rest)
    ent = ls + rest * 0.65625 / (1 + rest)
    tol = U * (4 * 0.65625 + 2 * (512 + 64) + 32)
    assert (got.logprobs.double() + ls).abs().max().item() <= tol + 4 * U * ls
    assert (got.entropy.double() - ent).abs().max().item() <= tol * (1 + ent)
    assert torch.equal(got.top_ids[:, 0], tok) and torch.equal(got.top_logprobs[:, 0], got.logprobs)
    del x
    torch.cuda.empty_cache()


def test_sizes_past_the_library_counts_are_refused(pkg, cuda):
    """2^32 + 43 columns are not 43, nor as many matrix columns 43."""
    torch = _torch()
    torch.cuda.empty_cache()
    x = torch.empty((1, (1 << 32) + 43), dtype=torch.float16, device=cuda)
    tok = torch.zeros(1, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="logits: at most"):
        pkg.policy.token_logprobs(x, tok)
    with pytest.raises(ValueError, match="logits: at most"):
        pkg.policy.token_logprobs_backward(x, tok, torch.zeros(1, 3, device=cuda))
    with pytest.raises(ValueError, match="g: at most"):
        pkg.policy.orthogonalize(x, out=x)
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,rows,vocab", [("f32", 300, 43), ("bf16", 3, 60001), ("f16", 16500, 42)])
def test_in_place_from_a_graph(pkg, cuda, dtype, rows, vocab):
    """Scores and the gradient in their place, captured and replayed on new logits between eager work."""
    torch = _torch()
    pol = pkg.policy
    x, tok = make(cuda, dtype, rows, vocab, ld=vocab + 1, seed=41)
    buf = torch.full((rows, vocab + 1), 9.0, dtype=x.dtype, device=cuda)
    y = buf[:, :vocab]
    g = torch.randn(rows, generator=torch.Generator().manual_seed(4)).to(cuda)

    def both(t, out):
        r = pol.token_logprobs(t, tok, stats=True)
        pol.token_logprobs_backward(t, tok, r.stats, g_logprobs=g, g_entropy=g, out=out)
        return r.logprobs

    y.copy_(x)
    both(y, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lp = both(y, y)
    for rep in range(4):
        x, _ = make(cuda, dtype, rows, vocab, ld=vocab + 1, seed=42 + rep)
        want = torch.empty_like(y)
        want_lp = both(x, want)
        y.copy_(x)
        lp.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(lp, want_lp) and buf[:, vocab].eq(9).all()
