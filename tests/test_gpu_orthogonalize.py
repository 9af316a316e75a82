"""cfp_orthogonalize / cfp_muon_update against the same products in 64 bits.

Tolerances (2-norm of the difference over that of the result).  A relative error d made in a
step's X or in its products reaches the result multiplied by at most the remaining steps' slopes
where singular values are small, and by about 1 where they have settled; relative to the norm
the whole is at most a few d per step.  With 5 steps and four roundings each (X, A, B, X'):
  three products: d = 2^-22 (what hi + lo and the left-out lo lo lose, halves of 2^-21) plus the
    fp32 accumulation, 2^-24 sqrt(K) for sums of K terms: 20 * 2^-22 + 20 * 2^-24 sqrt(K)
    <= 4.8e-6 + 1.2e-6 sqrt(K) / 1 -> taken as 5e-6 + 2^-22 sqrt(K) * 2
  one product: d = 2^-12 (half a step of fp16, 11 bits): 20 * 2^-12 = 4.9e-3
and the output's own rounding, eps / 2 of its type at most, on top."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

QUINTIC = (3.4445, -4.7750, 2.0315)
DT = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


def _torch():
    import torch
    return torch


def reference(g, steps=5, coefs=QUINTIC, eps=1e-7):
    """float64 on the CPU, [batch][rows][cols]."""
    torch = _torch()
    x = g.double().cpu()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    c = np.broadcast_to(np.asarray(coefs, dtype=np.float32).astype(np.float64), (steps, 3))
    for i in range(steps):
        a = x @ x.transpose(-1, -2)
        x = c[i][0] * x + (c[i][1] * a + c[i][2] * (a @ a)) @ x
    return x.transpose(-1, -2) if tall else x


def gradient(cuda, batch, rows, cols, dtype="f32", seed=0, fall=0.5, size=1e-3):
    """Sums of outer products with weights falling as 1 / k^fall."""
    torch = _torch()
    g = torch.Generator(device="cpu").manual_seed(seed)
    r = min(rows, cols)
    w = torch.arange(1, r + 1).float() ** -fall
    m = (torch.randn(batch, rows, r, generator=g) * w) @ torch.randn(batch, r, cols, generator=g) * size
    return m.to(getattr(torch, DT[dtype])).to(cuda)


def tolerance(dtype, products, shape):
    torch = _torch()
    k = max(shape[-2:])
    own = 4.9e-3 if products == 1 else 5e-6 + 2.0 ** -21 * np.sqrt(k)
    return own + torch.finfo(getattr(torch, DT[dtype])).eps / 2


def grown(g, steps=5):
    """Bound for spectra that leave most directions empty.  There the argument above does not
    hold: the result's norm is that of the few directions in use, while roundings fall into all
    of them and grow by the slope at zero, 3.4445, a step.  A rounding of X, A, B or of the products
    changes X_t by at most 2^-23 |X_t| (half a step of hi + lo's 22 bits), four of them a step:
      |error| <= sum_t 4 * 2^-23 |X_t| 3.4445^(steps - t)
    For a rank-one G (|X_t| about 1): 4 * 2^-23 * 683 = 3.3e-4.  An fp32 evaluation on the CPU
    is 2.7e-5 off for the spectrum 1 / k^3 below; this kernel 2.0e-5."""
    x = [reference(g, t) for t in range(steps + 1)]
    return sum(4 * 2.0 ** -23 * x[t].norm() * QUINTIC[0] ** (steps - t) for t in range(steps)).item() / x[-1].norm().item()


def off(got, want):
    d = (got.double().cpu() - want).flatten(1).norm(dim=1) if got.dim() == 3 else (got.double().cpu() - want).norm()
    n = want.flatten(1).norm(dim=1) if got.dim() == 3 else want.norm()
    return (d / n.clamp(min=1e-300)).max().item()


SHAPES = [(1, 1, 1), (1, 1, 7), (1, 9, 1), (2, 3, 5), (1, 31, 33), (3, 64, 64), (1, 65, 64), (1, 63, 130), (9, 256, 256),
          (1, 843, 256), (1, 256, 843), (2, 300, 1000), (1, 1000, 2731), (1, 2050, 700), (1, 40, 5000),
          (1, 128, 128), (2, 192, 700), (40, 250, 256), (3, 130, 3000), (1, 64, 9000), (1, 500, 4500),
          (300, 32, 32), (2, 64, 256), (3, 256, 61), (2, 97, 100), (1, 20, 500), (1, 128, 126),
          (1, 500, 1000), (4, 256, 843)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,rows,cols", SHAPES)
def test_against_64_bits(pkg, cuda, dtype, batch, rows, cols):
    g = gradient(cuda, batch, rows, cols, dtype, seed=rows + cols)
    want = reference(g)
    for products in (0, 1, 3):
        got = pkg.policy.orthogonalize(g, products=products)
        assert got.shape == g.shape and got.dtype == g.dtype
        used = products or (1 if dtype == "bf16" else 3)
        assert off(got, want) <= tolerance(dtype, used, g.shape), (products, off(got, want))


def test_spectra(pkg, cuda):
    """Flat, falling and single-direction spectra; the singular values that come out."""
    torch = _torch()
    for fall in (0.0, 1.0, 3.0):
        g = gradient(cuda, 1, 200, 320, seed=3, fall=fall)
        assert off(pkg.policy.orthogonalize(g), reference(g)) <= (grown(g) if fall == 3.0 else tolerance("f32", 3, g.shape))
    u, v = torch.randn(1, 150, 1, device=cuda), torch.randn(1, 1, 90, device=cuda)
    g = u * v
    got = pkg.policy.orthogonalize(g)
    assert off(got, reference(g)) <= grown(g)
    # every singular value is the polynomial of the input's: one below 0.6 / 3.4445^5 = 1.2e-3 of
    # |G| cannot have reached the band of 0.68 .. 1.21 that the others end in
    g = gradient(cuda, 1, 128, 256, fall=0.0)
    s = torch.linalg.svdvals(pkg.policy.orthogonalize(g)[0].double().cpu())
    x = torch.linalg.svdvals(g[0].double().cpu()) / g.double().cpu().norm()
    start = x
    for _ in range(5):
        x = QUINTIC[0] * x + QUINTIC[1] * x ** 3 + QUINTIC[2] * x ** 5
    assert (s.sort()[0] - x.sort()[0]).norm() <= tolerance("f32", 3, g.shape) * x.norm()
    reached = x[start > 2e-3]
    assert reached.min() > 0.6 and s.max() < 1.25


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 8, 16])
def test_step_counts_and_coefficients(pkg, cuda, steps):
    torch = _torch()
    g = gradient(cuda, 2, 70, 150, seed=steps)
    assert off(pkg.policy.orthogonalize(g, steps=steps), reference(g, steps)) <= tolerance("f32", 3, g.shape) * max(1, steps / 5)
    assert off(pkg.policy.orthogonalize(g, steps=steps, coefs=(1.875, -1.25, 0.375)),
               reference(g, steps, (1.875, -1.25, 0.375))) <= tolerance("f32", 3, g.shape) * max(1, steps / 5)
    if steps:
        cs = np.linspace(0, 1, steps)[:, None] * np.array([[-0.5, 0.3, -0.1]]) + np.array(QUINTIC)
        assert off(pkg.policy.orthogonalize(g, steps=steps, coefs=cs), reference(g, steps, cs)) <= tolerance("f32", 3, g.shape) * max(1, steps / 5)


def test_sizes_of_values(pkg, cuda):
    """Squares that would overflow or vanish in 32 bits, a norm below eps, zeros, NaN, infinity."""
    torch = _torch()
    base = gradient(cuda, 1, 48, 80, seed=2, size=1.0)
    for size in (1e30, 1e-4, 1e-30, 1e-38):
        g = base * size
        assert off(pkg.policy.orthogonalize(g, eps=0.0), reference(g, eps=0.0)) <= tolerance("f32", 3, g.shape)
    small = base * 1e-9                    # |G| of the order of eps: not yet normalised, still right
    assert off(pkg.policy.orthogonalize(small), reference(small)) <= tolerance("f32", 3, base.shape)
    assert pkg.policy.orthogonalize(torch.zeros(2, 30, 50, device=cuda)).eq(0).all()
    assert pkg.policy.orthogonalize(torch.zeros(2, 30, 50, device=cuda), eps=0.0).eq(0).all()
    g = torch.cat([base, base])
    g[1, 5, 7] = float("nan")
    got = pkg.policy.orthogonalize(g)
    assert got[1].isnan().all() and not got[0].isnan().any()
    g[1, 5, 7] = float("inf")
    assert pkg.policy.orthogonalize(g)[1].isnan().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [(90, 200), (200, 90)])
def test_strides_offsets_and_in_place(pkg, cuda, dtype, rows, cols):
    torch = _torch()
    g = gradient(cuda, 3, rows, cols, dtype, seed=7)
    want = pkg.policy.orthogonalize(g)
    store = torch.full((1 + 3 * (rows + 2) * (cols + 3),), 5.0, dtype=g.dtype, device=cuda)
    view = store[1:].view(3, rows + 2, cols + 3)[:, 1:1 + rows, 2:2 + cols]
    view.copy_(g)
    before = store.clone()
    out = torch.full((3, rows + 1, cols + 5), 6.0, dtype=g.dtype, device=cuda)
    got = pkg.policy.orthogonalize(view, out=out[:, :rows, 3:3 + cols])
    assert torch.equal(got, want) and torch.equal(store, before)
    assert out[:, rows:].eq(6).all() and out[:, :, :3].eq(6).all() and out[:, :, 3 + cols:].eq(6).all()
    pkg.policy.orthogonalize(view, out=view)
    assert torch.equal(view, want)
    mask = torch.ones_like(store, dtype=torch.bool)
    mask[1:].view(3, rows + 2, cols + 3)[:, 1:1 + rows, 2:2 + cols] = False
    assert store[mask].eq(5).all()
    assert torch.equal(pkg.policy.orthogonalize(g[1]), want[1])       # a batch changes nothing


def muon_reference(w, g, m, lr, beta, nesterov, decay, scale):
    w, g, m = w.double().cpu(), g.double().cpu(), m.double().cpu()
    m = beta * m + g
    o = reference(g + beta * m if nesterov else m)
    rows, cols = w.shape[-2:]
    scale = scale or max(1.0, rows / cols) ** 0.5
    return w * (1 - lr * decay) - lr * scale * o, m, lr * scale * o


@pytest.mark.parametrize("products", [1, 3])
@pytest.mark.parametrize("batch,rows,cols", [(9, 256, 256), (1, 843, 256), (2, 33, 70), (1, 700, 1500)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(pkg, cuda, batch, rows, cols, nesterov, products):
    torch = _torch()
    w = gradient(cuda, batch, rows, cols, seed=1, size=0.1)
    m = gradient(cuda, batch, rows, cols, seed=2)
    for it in range(2):
        g = gradient(cuda, batch, rows, cols, seed=3 + it)
        keep = g.clone()
        want_w, want_m, step = muon_reference(w, g, m, 0.02, 0.95, nesterov, 0.1, 0.0)
        lr = 0.02 if it == 0 else torch.tensor([0.02], device=cuda)
        pkg.policy.muon_update(w, g, m, lr, nesterov=nesterov, weight_decay=0.1, products=products)
        assert torch.equal(g, keep)
        assert off(m, want_m) <= 2.0 ** -23
        # the weight's own roundings (three) and the step's error
        d = (w.double().cpu() - want_w).flatten(1).norm(dim=1)
        bound = tolerance("f32", products, w.shape) * step.flatten(1).norm(dim=1) + 3 * 2.0 ** -24 * want_w.flatten(1).norm(dim=1)
        assert (d <= bound).all()


def test_muon_scale_and_strides(pkg, cuda):
    torch = _torch()
    big = [torch.full((3, 50, 64), 4.0, device=cuda) for _ in range(3)]
    w, g, m = (t[:, 5:45, 8:48] for t in big)
    for i, t in enumerate((w, g, m)):
        t.copy_(gradient(cuda, 3, 40, 40, seed=i))
    want_w, want_m, step = muon_reference(w, g, m, 0.5, 0.9, True, 0.0, 0.2)
    pkg.policy.muon_update(w, g, m, 0.5, momentum=0.9, scale=0.2)
    assert off(m, want_m) <= 2.0 ** -23
    assert (w.double().cpu() - want_w).norm() <= tolerance("f32", 3, w.shape) * step.norm() + 2.0 ** -22 * want_w.norm()
    for t in big:
        assert t[:, :5].eq(4).all() and t[:, 45:].eq(4).all() and t[:, :, :8].eq(4).all() and t[:, :, 48:].eq(4).all()


def test_same_call_same_bits_on_any_stream_and_from_a_graph(pkg, cuda):
    torch = _torch()
    pol = pkg.policy
    for dtype, shape in (("f32", (9, 256, 256)), ("bf16", (1, 700, 1300)), ("f32", (1, 300, 80))):
        g = gradient(cuda, *shape, dtype, seed=5)
        want = pol.orthogonalize(g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(pol.orthogonalize(g), want)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        w, m = torch.zeros(shape, device=cuda), torch.zeros(shape, device=cuda)
        lr = torch.tensor([0.1], device=cuda)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = pol.orthogonalize(g)
            pol.muon_update(w, g.float(), m, lr)
        w2, m2 = torch.zeros_like(w), torch.zeros_like(m)
        for rep in range(3):
            g.copy_(gradient(cuda, *shape, dtype, seed=20 + rep))
            lr.fill_(0.1 / (rep + 1))
            eager = pol.orthogonalize(g)
            pol.muon_update(w2, g.float(), m2, 0.1 / (rep + 1))
            out.fill_(3)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and torch.equal(m, m2)
            assert (w - w2).abs().max().item() <= 2.0 ** -20


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(300, 40, 60), (5, 64, 256), (2, 500, 330)])
def test_small_matrices_from_a_graph_in_place_and_side_by_side(pkg, cuda, dtype, shape):
    """One workgroup a matrix and many: captured and replayed, in place, columns beside the input's."""
    torch = _torch()
    pol = pkg.policy
    batch, rows, cols = shape
    g = gradient(cuda, *shape, dtype, seed=11)
    wide = torch.full((batch, rows, 2 * cols + 1), 3.0, dtype=g.dtype, device=cuda)
    wide[:, :, 1:cols + 1].copy_(g)
    want = pol.orthogonalize(g)
    pol.orthogonalize(wide[:, :, 1:cols + 1], out=wide[:, :, cols + 1:])
    assert torch.equal(wide[:, :, cols + 1:], want) and torch.equal(wide[:, :, 1:cols + 1], g) and wide[:, :, 0].eq(3).all()
    buf = g.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pol.orthogonalize(buf, out=buf)
    for rep in range(4):
        g = gradient(cuda, *shape, dtype, seed=30 + rep)
        buf.copy_(g)
        eager = pol.orthogonalize(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf, eager)
        assert off(buf, reference(g)) <= tolerance(dtype, 1 if dtype == "bf16" else 3, shape)


def test_arrays_packed_matrix_by_matrix(pkg, cuda):
    """Weights, gradients and momentum of a layer behind each other, and rows taken in turn."""
    torch = _torch()
    for shape in ((4, 3, 50, 70), (4, 50, 3, 70)):
        packed = torch.full(shape, 2.0, device=cuda)
        at = (lambda k: packed[:, k]) if shape[1] == 3 else (lambda k: packed[:, :, k])
        w, g, m = (at(k) for k in range(3))
        for i, t in enumerate((w, g, m)):
            t.copy_(gradient(cuda, 4, 50, 70, seed=40 + i))
        w2, g2, m2 = (t.contiguous().clone() for t in (w, g, m))
        pkg.policy.muon_update(w, g, m, 0.1)
        pkg.policy.muon_update(w2, g2, m2, 0.1)
        assert torch.equal(w, w2) and torch.equal(g, g2) and torch.equal(m, m2)


def test_two_calls_at_once(pkg, cuda):
    """Two streams, each call with a workspace of its own."""
    torch = _torch()
    gs = [gradient(cuda, 1, 512, 900, seed=i) for i in range(2)]
    want = [pkg.policy.orthogonalize(g) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(pkg.policy.orthogonalize(gs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, want[i])


def test_refusals_with_device_tensors(pkg, cuda):
    torch = _torch()
    pol = pkg.policy
    g = torch.zeros(8, 12, device=cuda)
    for bad in (lambda: pol.orthogonalize(g.double()), lambda: pol.orthogonalize(g[0]), lambda: pol.orthogonalize(g.t()),
                lambda: pol.orthogonalize(g, out=torch.zeros(8, 11, device=cuda)),
                lambda: pol.orthogonalize(g[:0]),
                lambda: pol.muon_update(g, g.clone().bfloat16(), g.clone(), 0.1),
                lambda: pol.muon_update(g, g.clone(), torch.zeros(8, 13, device=cuda)[:, :12], 0.1),
                lambda: pol.muon_update(g.bfloat16(), g.bfloat16(), g.bfloat16(), 0.1),
                lambda: pol.muon_update(g, g.clone(), g.clone(), torch.zeros(2, device=cuda)),
                lambda: pol.muon_update(g, g.clone(), g.clone(), torch.zeros(1))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(pkg._lib.CfpError, match="steps"):
        pol.orthogonalize(g, steps=17)
    with pytest.raises(pkg._lib.CfpError, match="overlap"):
        pol.orthogonalize(g[None].expand(3, 8, 12))
    assert pol.orthogonalize(torch.zeros(0, 4, 4, device=cuda)).numel() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("batch,rows,cols", [(1, 31, 33), (1, 128, 128), (9, 256, 256), (1, 256, 843), (2, 192, 700),
                                             (1, 2050, 700), (1, 1024, 1024), (1, 64, 9000)])
def test_fewer_bits_only_when_asked_for(pkg, cuda, dtype, batch, rows, cols):
    """By default every type gets the accuracy of fp32 and one rounding to its own at the end.  With
    e the error before that rounding, nearest(w + e) is at most |nearest(w) - w| + 2 |e| from w."""
    torch = _torch()
    g = gradient(cuda, batch, rows, cols, dtype, seed=3 * rows + cols)
    want = reference(g)
    once = off(want.to(g.dtype), want)
    got = pkg.policy.orthogonalize(g)
    assert off(got, want) <= once + 2 * (5e-6 + 2.0 ** -21 * np.sqrt(max(rows, cols))), (off(got, want), once)
    assert torch.equal(got, pkg.policy.orthogonalize(g, products=3))


@pytest.mark.parametrize("outputs,inputs", [(300, 80), (80, 300), (843, 256)])
def test_default_scale_is_that_of_outputs_by_inputs(pkg, cuda, outputs, inputs):
    """The step of a weight stored the other way round is the transposed one, its factor given."""
    torch = _torch()
    w, g, m = (gradient(cuda, 1, outputs, inputs, seed=50 + k, size=0.1 if k == 0 else 1e-3) for k in range(3))
    w2, g2, m2 = (t.transpose(1, 2).contiguous() for t in (w, g, m))
    want, _, step = muon_reference(w, g, m, 0.1, 0.95, True, 0.0, max(1.0, outputs / inputs) ** 0.5)
    pkg.policy.muon_update(w, g, m, 0.1)
    pkg.policy.muon_update(w2, g2, m2, 0.1, scale=max(1.0, outputs / inputs) ** 0.5)
    bound = tolerance("f32", 3, w.shape) * step.norm() + 3 * 2.0 ** -24 * want.norm()
    assert (w.double().cpu() - want).norm() <= bound
    assert (w2.transpose(1, 2).double().cpu() - want).norm() <= bound


@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("rows,cols", [(30, 50), (300, 90)])
def test_nan_and_infinity_take_the_whole_matrix(pkg, cuda, rows, cols, steps):
    """At any number of steps, none among them; the batch's other matrices keep their values."""
    torch = _torch()
    base = gradient(cuda, 3, rows, cols, seed=8)
    want = pkg.policy.orthogonalize(base, steps=steps)
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = base.clone()
        g[1, rows - 1, 3] = bad
        got = pkg.policy.orthogonalize(g, steps=steps)
        assert got[1].isnan().all() and torch.equal(got[::2], want[::2])
    assert pkg.policy.orthogonalize(base, steps=steps, eps=float("inf")).eq(0).all()


@pytest.mark.parametrize("rows,cols", [(48, 80), (256, 300), (900, 700)])
@pytest.mark.parametrize("below", [1.0, 1e3, 1e6, 1e9])
def test_norms_far_below_eps(pkg, cuda, rows, cols, below):
    """|G| = eps / below.  X is held to 2^-35 an entry (half a denormal step of fp16, times 2^10), so
    every step leaves up to 2^-35 sqrt(rows cols), which the remaining ones amplify by 3.4445 each at
    most: 683 times that (the sum of the powers 1 .. 5).  A and B are held to 2^-33: (4.775 + 1) 2^-33 m
    of X a step."""
    g = gradient(cuda, 1, rows, cols, seed=rows)
    g *= 1e-7 / below / g.norm()
    want = reference(g)
    got = pkg.policy.orthogonalize(g)
    m = min(rows, cols)
    bound = (tolerance("f32", 3, g.shape) + 5 * 5.775 / 3.4445 * 2.0 ** -33 * m) * want.norm() + 683 * 2.0 ** -35 * (rows * cols) ** 0.5
    assert (got.double().cpu() - want).norm() <= bound


def in_the_formats(g, products, steps=5, eps=1e-7):
    """The definition with the kernels' number formats, on the CPU: X, A and B as fp16 (scaled by 2^10,
    2^8, 2^8) or hi + lo pairs of it, products hi hi (+ hi lo + lo hi), sums in float32 of another order."""
    torch = _torch()

    def pair(v, scale):
        v = (v * scale).float()
        hi = v.half().float()
        return hi / scale, (v - hi).half().float() / scale

    def product(l, r):
        out = l[0] @ r[0]
        return out if products == 1 else out + (l[0] @ r[1] + l[1] @ r[0])

    x = g.double().cpu()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = (x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)).float()
    turned = lambda p: tuple(t.transpose(-1, -2).contiguous() for t in p)
    for _ in range(steps):
        X = pair(x, 1024.0)
        A = pair(product(X, turned(X)), 256.0)
        a = A[0] if products == 1 else A[0] + A[1]
        B = pair(QUINTIC[1] * a + QUINTIC[2] * product(A, A), 256.0)
        x = QUINTIC[0] * (X[0] + X[1]) + product(B, X)
    return (x.transpose(-1, -2) if tall else x).double()


@pytest.mark.parametrize("products", [1, 3])
@pytest.mark.parametrize("rows,cols,fall", [(200, 320, 0.0), (200, 320, 1.0), (200, 320, 3.0), (60, 90, 0.5), (843, 256, 0.5),
                                            (700, 900, 0.5), (128, 512, 0.5), (1, 300, 0.0), (150, 400, None)])
def test_errors_are_those_of_the_formats(pkg, cuda, products, rows, cols, fall):
    """Against 64 bits the kernels are off by what their number formats leave, measured by the same
    roundings on the CPU rather than bounded.  One product: fp16's roundings (2^-12) are the same on
    both sides but where sums in fp32, off by up to 2^-24 sqrt(K) of themselves, fall on the other
    side of a border; that happens to a part 2^-13 sqrt(K) of them and moves those by a step, 12
    times a rounding's square: sqrt(12 * 2^-13 * sqrt(1024)) = 0.22 of the roundings' norm, taken as
    half of it.  Three: the 2^-23 of the pairs and the fp32 sums weigh alike, and sums are formed in
    another order, sixteen terms at a time here: taken as up to three times the norm.  fall None: one
    direction only."""
    torch = _torch()
    if fall is None:
        gen = torch.Generator().manual_seed(3)
        g = (torch.randn(1, rows, 1, generator=gen) * torch.randn(1, 1, cols, generator=gen)).to(cuda)
    else:
        g = gradient(cuda, 1, rows, cols, seed=rows + 5, fall=fall)
    want = reference(g)
    there = (in_the_formats(g, products) - want).norm()
    here = (pkg.policy.orthogonalize(g, products=products).double().cpu() - want).norm()
    assert here <= (1.5 if products == 1 else 3.0) * there + 2.0 ** -24 * want.norm(), (here / want.norm(), there / want.norm())


@pytest.mark.parametrize("batch,rows,cols", [(1, 65536, 1), (1, 1, 65536), (1, 65536, 40), (1, 200, 65536)])
def test_largest_sides_and_batches(pkg, cuda, batch, rows, cols):
    g = gradient(cuda, batch, rows, cols, seed=12, fall=0.0)
    got = pkg.policy.orthogonalize(g)
    assert off(got, reference(g)) <= tolerance("f32", 3, g.shape)
    assert off(pkg.policy.orthogonalize(g, products=1), reference(g)) <= tolerance("f32", 1, g.shape)


@pytest.mark.parametrize("products", [1, 3])
def test_the_largest_batch(pkg, cuda, products):
    """65 535 random matrices of 3 x 2.  Among so many some are nearly of one direction, and the bound is
    grown()'s for each: four roundings a step, of 2^-23 (three products) or 2^-12 (one) of X, amplified by
    3.4445 a step that follows.  (tolerance() holds for matrices that use all their directions alike.)"""
    g = gradient(cuda, 65535, 3, 2, seed=12, fall=0.0)
    x = [reference(g, t).flatten(1).norm(dim=1) for t in range(5)]
    bound = sum(4 * 2.0 ** (-12 if products == 1 else -23) * x[t] * QUINTIC[0] ** (5 - t) for t in range(5))
    error = (pkg.policy.orthogonalize(g, products=products).double().cpu() - reference(g)).flatten(1).norm(dim=1)
    assert (error <= bound).all(), (error / bound).max().item()
    assert error.median() <= tolerance("f32", products, g.shape)


@pytest.mark.parametrize("cols", [50, 400])
def test_rows_far_apart(pkg, cuda, cols):
    """Rows 2^30 + 9 entries apart: the third begins 2^33 bytes in."""
    torch = _torch()
    torch.cuda.empty_cache()
    ld = (1 << 30) + 9
    small = [gradient(cuda, 1, 3, cols, seed=60 + k)[0] for k in range(3)]
    want_o = pkg.policy.orthogonalize(small[1])
    store = torch.empty(3 * ld, device=cuda)
    at = lambda k: torch.as_strided(store, (3, cols), (ld, 1), k * cols)
    for k in range(3):
        at(k).copy_(small[k])
    pkg.policy.orthogonalize(at(1), out=at(3))
    assert torch.equal(at(3), want_o)
    pkg.policy.muon_update(*(at(k) for k in range(3)), 0.1)
    pkg.policy.muon_update(*small, 0.1)
    for k in range(3):
        assert torch.equal(at(k), small[k])
    del store
    torch.cuda.empty_cache()


def test_many_matrices_that_need_a_workspace(pkg, cuda):
    """20 000 matrices of 128 x 160: the first, the middle and the last as in 64 bits, in the batch's plan."""
    torch = _torch()
    torch.cuda.empty_cache()
    few = gradient(cuda, 3, 128, 160, seed=70)
    g = few.repeat(6667, 1, 1)[:20000]
    got = pkg.policy.orthogonalize(g)
    want = reference(few)
    for k in (0, 10000, 19999):
        assert off(got[k], want[k % 3]) <= tolerance("f32", 3, few.shape)
    assert torch.equal(got[:3].repeat(6667, 1, 1)[:20000], got)
    del g, got
    torch.cuda.empty_cache()
