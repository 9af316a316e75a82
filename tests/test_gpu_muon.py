"""The trainer's Muon optimiser (cfp_train_set_optimizer, cfp_train_muon, cfp_train_update with it)
and the new operators in the order a training program uses them: forward, scores of the taken
actions, their gradient, weight gradients, orthogonalised step."""
import numpy as np
import pytest

from parity_util import ACTIONS, GRU, HIDDEN, OBS, synth_records_host
from test_gpu_orthogonalize import grown, off, reference, tolerance
from test_gpu_train import _collect, _segments, _t

pytestmark = pytest.mark.gpu


def _expected(before, g, mom, lr, wd, beta, nesterov):
    """(W_enc, W_gru) after one step in float64, the step sizes, and the new momenta."""
    import torch
    out = {}
    for name, shape in (("W_enc", (1, OBS, HIDDEN)), ("W_gru", (-1, HIDDEN, HIDDEN))):
        w, gr, m = (torch.from_numpy(a[name]).double().reshape(shape) for a in (before, g, mom))
        m = beta * m + gr
        u = gr + beta * m if nesterov else m
        step = lr * reference(u)
        out[name] = (w * (1 - lr * wd) - step, step, m, u)
    return out


@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("bf16", [False, True])
def test_steps_against_64_bits(pkg, cuda, layers, nesterov, bf16):
    """Two steps with random gradients: matrices as cfp_muon_update's definition, everything else
    as a twin's Adam, bit for bit; the grads arena ends as zeros."""
    import torch
    rng = np.random.default_rng(5)
    pols = [pkg.Policy(64, layers, seed=21) for _ in range(2)]
    trs = [pkg.Trainer(p, 4) for p in pols]
    trs[0].set_optimizer("muon", lr=0.05, weight_decay=0.1, momentum=0.9, nesterov=int(nesterov))
    assert trs[0].optimizer == "muon" and trs[1].optimizer == "adam"
    if bf16:
        trs[0].set_gemm_mode(bf16=1)
    mom = {n: np.zeros(s.stop - s.start, np.float32) for n, s in _segments(layers)}
    for it in range(2):
        before = pols[0].get_params()
        parts = {n: before[s] for n, s in _segments(layers)}
        g = (rng.standard_normal(before.size) * 0.1).astype(np.float32)
        want = _expected(parts, {n: g[s] for n, s in _segments(layers)}, mom, 0.05, 0.1, 0.9, nesterov)
        for tr in trs:
            tr.buf("grads").copy_(_t(g, cuda))
        trs[0].muon(); trs[1].adam()
        torch.cuda.synchronize()
        after, twin = pols[0].get_params(), pols[1].get_params()
        assert not trs[0].buf("grads").any()
        arena_m = trs[0].buf("adam_m").cpu().numpy()
        for n, s in _segments(layers):
            if n not in want:
                assert np.array_equal(after[s], twin[s]), n
                continue
            w, step, m, u = want[n]
            got = torch.from_numpy(after[s]).double().reshape(w.shape)
            err = (got - w).flatten(1).norm(dim=1)
            # 0.05 * the polar factor's error + three roundings of the weight
            bound = tolerance("f32", 1 if bf16 else 3, w.shape) * step.flatten(1).norm(dim=1) + 3 * 2.0 ** -24 * w.flatten(1).norm(dim=1)
            assert (err <= bound).all(), (n, it)
            mom[n] = arena_m[s]
            gm = torch.from_numpy(arena_m[s]).double().reshape(m.shape)
            assert (gm - m).norm() <= 2.0 ** -23 * m.norm()
    for tr, p in zip(trs, pols):
        tr.close(); p.close()


def test_step_writes_every_weight_mirror(pkg, cuda):
    """As the Adam step does: after a step the forwards equal those of a fresh policy that got the
    same parameters, in fp32 (both tile sizes) and with bf16 inputs."""
    import torch
    n, layers = 64, 3
    pol = pkg.Policy(n, layers, seed=21)
    tr = pkg.Trainer(pol, 4)
    tr.set_optimizer("muon")
    rng = np.random.default_rng(22)
    before = pol.get_params()
    for _ in range(2):
        tr.buf("grads").copy_(_t((rng.standard_normal(before.size) * 0.1).astype(np.float32), cuda))
        tr.muon()
    torch.cuda.synchronize()
    after = pol.get_params()
    assert np.mean(after != before) > 0.999
    twin = pkg.Policy(n, layers, seed=99)
    twin.set_params(after)
    rec = _t(synth_records_host(n, 23, 0), cuda)
    term = torch.zeros(n, device=cuda)
    s0 = (0.5 * rng.standard_normal((layers, n, HIDDEN))).astype(np.float32)
    for bf16, small in ((False, False), (True, False), (False, True)):
        for p in (pol, twin):
            p.set_gemm_bf16(bf16); p.set_small_tiles(small)
        sa, sb = _t(s0, cuda), _t(s0, cuda)
        assert torch.equal(pol.forward(rec, term, sa), twin.forward(rec, term, sb)), (bf16, small)
        assert torch.equal(sa, sb)
    tr.close(); pol.close(); twin.close()


@pytest.mark.parametrize("on_side_stream", [False, True])
def test_update_eager_and_graph_match_the_manual_loop(pkg, cuda, on_side_stream):
    """cfp_train_update with Muon, eager and replayed, against the loop written out; both learning
    rates change between iterations through their device scalars."""
    import torch
    n, T = 64, 6
    cfg = dict(epochs=2, minibatches=2)
    trip = [_collect(pkg, cuda, n, T, 321, 0.1, **cfg) for _ in range(3)]
    (_, pol_m, tr_m, _), (_, pol_e, tr_e, _), (_, pol_g, tr_g, _) = trip
    mb = n // 2
    stream = torch.cuda.Stream() if on_side_stream else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        for tr in (tr_m, tr_e, tr_g):
            tr.set_optimizer("muon", lr=0.01)
        for it in range(3):
            for tr in (tr_m, tr_e, tr_g):
                tr.buf("lr").fill_(3e-4 * (1.0 - 0.25 * it))
                tr.buf("muon_lr").fill_(0.01 * (1.0 - 0.25 * it))
            for _ in range(cfg["epochs"]):
                tr_m.zero_loss()
                for m in range(cfg["minibatches"]):
                    tr_m.backward(m * mb, mb)
                    tr_m.muon()
            tr_e.update(use_graph=False)
            tr_g.update(use_graph=True)
            torch.cuda.synchronize()
            assert np.isfinite(torch.randn(1 << 16, device=cuda).sum().item())   # eager work between replays
            for name, pol, tr in (("eager", pol_e, tr_e), ("graph", pol_g, tr_g)):
                assert torch.equal(pol.params, pol_m.params), f"{name} params, iteration {it}"
                for b in ("adam_m", "adam_v", "loss_acc"):
                    assert torch.equal(tr.buf(b), tr_m.buf(b)), f"{name} {b} {it}"
                assert not tr.buf("grads").any()
        # another configuration, and Adam again: the next graph calls capture anew
        for kind, kw in (("muon", dict(lr=0.005, momentum=0.8, steps=3)), ("adam", {})):
            for tr in (tr_m, tr_g):
                tr.set_optimizer(kind, **kw)
            for _ in range(cfg["epochs"]):
                tr_m.zero_loss()
                for m in range(cfg["minibatches"]):
                    tr_m.backward(m * mb, mb)
                    tr_m.muon() if kind == "muon" else tr_m.adam()
            tr_g.update(use_graph=True)
            torch.cuda.synchronize()
            assert torch.equal(pol_g.params, pol_m.params), kind
    for _, pol, tr, _ in trip:
        tr.close(); pol.close()


def test_change_of_optimizer_starts_the_moments_anew(pkg, cuda):
    """Adam -> Muon -> Adam: the second Adam is a fresh trainer's, bit for bit; setting the same
    kind again keeps the moments."""
    import torch
    pols = [pkg.Policy(32, 1, seed=4) for _ in range(2)]
    a, b = (pkg.Trainer(p, 2) for p in pols)
    g = torch.randn(pols[0].param_count, device=cuda)
    a.buf("grads").copy_(g); a.adam()
    a.set_optimizer("muon"); a.buf("grads").copy_(g); a.muon()
    a.set_optimizer("muon", lr=0.5)
    torch.cuda.synchronize()
    assert a.buf("adam_m").any() and a.buf("muon_lr").item() == 0.5
    a.set_optimizer("adam")
    torch.cuda.synchronize()
    assert not a.buf("adam_m").any() and not a.buf("adam_v").any()
    pols[0].set_params(pols[1].get_params())
    for t in (a, b):
        t.buf("grads").copy_(g); t.adam()
    torch.cuda.synchronize()
    assert torch.equal(pols[0].params, pols[1].params) and torch.equal(a.buf("adam_v"), b.buf("adam_v"))
    with pytest.raises(pkg._lib.CfpError, match="optimiser is Adam"):
        a.muon()
    with pytest.raises(pkg._lib.CfpError, match="steps"):
        a.set_optimizer("muon", steps=17)
    with pytest.raises(pkg._lib.CfpError, match="momentum"):
        a.set_optimizer("muon", momentum=1.0)
    with pytest.raises(ValueError):
        a.set_optimizer("sgd")
    assert a.optimizer == "adam"
    for t, p in zip((a, b), pols):
        t.close(); p.close()


def test_the_operators_as_a_training_step_uses_them(pkg, cuda):
    """Policy gradient of the actor head through the public calls: forward (heads, top layer's
    output), token_logprobs on the 43 logits of the 44-wide head rows, its gradient, dW by the GEMM
    seam, one Muon step; against the same chain in float64."""
    import torch
    n, layers = 512, 2
    pol = pkg.Policy(n, layers, seed=3)
    rec = pkg.policy.synth_records(n, 5, 1)
    h3 = torch.empty((n, HIDDEN), device=cuda)
    av = pol.forward(rec, torch.zeros(n, device=cuda), torch.zeros((layers, n, HIDDEN), device=cuda), h3=h3)
    act, _, _ = pkg.policy.value_sample(av, 9)
    adv = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(cuda)
    got = pkg.policy.token_logprobs(av[:, :ACTIONS], act, top=3, stats=True)
    g_lp, g_ent = -adv / n, torch.full((n,), -0.01 / n, device=cuda)
    dlogits = pkg.policy.token_logprobs_backward(av[:, :ACTIONS], act, got.stats, g_logprobs=g_lp, g_entropy=g_ent)
    dW = torch.zeros((ACTIONS, HIDDEN), device=cuda)
    pkg.policy.gemm_dw(h3, dlogits, dW)
    w = torch.from_numpy(pkg.policy.split_params(pol.get_params(), layers)["W_a"].copy()).to(cuda)
    w0, mom = w.clone(), torch.zeros_like(w)
    pkg.policy.muon_update(w, dW, mom, 0.02)
    # float64: logits from the same h3 and weights, loss by autograd
    W = w0.double().cpu().requires_grad_()
    b = torch.from_numpy(pkg.policy.split_params(pol.get_params(), layers)["b_a"].copy()).double()
    lp = torch.log_softmax(h3.double().cpu() @ W.T + b, 1)
    loss = (lp.gather(1, act.cpu().long()[:, None])[:, 0] * g_lp.double().cpu()).sum() + \
        (-(lp.exp() * lp).sum(1) * g_ent.double().cpu()).sum()
    grad, = torch.autograd.grad(loss, W)
    # the logits' own fp32 error (K = 256 sums) dominates: 1e-4 as everywhere in the GEMM tests
    assert (dW.double().cpu() - grad).norm() <= 1e-4 * grad.norm()
    # Against the update of the 64-bit gradient: a relative change d of the gradient moves the
    # polar factor by at most d |G| / (smallest singular value in use), through the polynomial's
    # slope of at most 3.4445^5 = 485 over |X_0| = 1: 485 * 1e-4 in the worst direction.  Against
    # the update of the gradient it was given, the operator's own tolerance holds.
    for g, tol in ((grad, 485 * 1e-4), (dW.double().cpu(), tolerance("f32", 3, dW.shape) + grown(dW))):
        o = 0.02 * reference(1.95 * g)
        assert ((w0.double().cpu() - o) - w.double().cpu()).norm() <= tol * o.norm() + 3 * 2.0 ** -24 * w0.double().cpu().norm()
    assert got.top_ids.shape == (n, 3) and (got.top_logprobs[:, :1] >= got.logprobs[:, None] - 1e-5).all()
    pol.close()


def test_an_adam_step_of_a_muon_trainer_is_refused(pkg, cuda):
    """Its first moment holds Muon's momentum: nothing may change."""
    import torch
    pol = pkg.Policy(32, 1, seed=4)
    tr = pkg.Trainer(pol, 2)
    tr.set_optimizer("muon")
    g = torch.randn(pol.param_count, device=cuda)
    tr.buf("grads").copy_(g)
    tr.muon()
    tr.buf("grads").copy_(g)
    before = pol.get_params(), tr.buf("adam_m").clone(), tr.buf("adam_v").clone()
    with pytest.raises(pkg._lib.CfpError, match="optimiser is Muon"):
        tr.adam()
    torch.cuda.synchronize()
    assert np.array_equal(pol.get_params(), before[0]) and torch.equal(tr.buf("grads"), g)
    assert torch.equal(tr.buf("adam_m"), before[1]) and torch.equal(tr.buf("adam_v"), before[2])
    tr.set_optimizer("adam")
    tr.buf("grads").copy_(g)
    tr.adam()
    torch.cuda.synchronize()
    assert not np.array_equal(pol.get_params(), before[0])
    tr.close(); pol.close()
