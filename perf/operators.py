"""Cases for the operators around a policy's distribution and its weights: log-probabilities
of given tokens (actions) with entropy and top alternatives, their gradient, and the
orthogonalised update of a weight matrix (Newton-Schulz products), alone and as a whole
optimiser step with momentum.

`run` with `own` false computes them from elementary torch operations; with `own` true it makes
the calls a user makes: policy.token_logprobs, policy.token_logprobs_backward,
policy.orthogonalize, policy.muon_update.
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
# coefficients of the odd quintic a x + b x^3 + c x^5 of the Muon optimiser's write-up
QUINTIC = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
MOMENTUM = 0.95
LR = 0.02
DECAY = 0.01


def _policy():
    import __graft_entry__ as entry
    return entry.load_package().policy


# ---- cases -------------------------------------------------------------------------------
def listed():
    return [
        # one rollout step's action rows straight from the fused head (44 floats wide: 43
        # logits and the value), re-evaluated under the current weights: latency counts
        dict(name="actions_step", op="logprobs", dtype="f32", rows=4096, vocab=43, ld=44, mask=0, top=0),
        # a whole stored rollout (4096 envs x 64 steps) with a mask of the allowed actions
        dict(name="actions_rollout", op="logprobs", dtype="f32", rows=262144, vocab=43, ld=44, mask=1, top=0),
        # one generated token of a language model: the smallest call over the widest row
        dict(name="token_one", op="logprobs", dtype="bf16", rows=1, vocab=131072, ld=131072, mask=0, top=20),
        # scoring a prompt, with alternatives: the largest read
        dict(name="tokens_prompt", op="logprobs", dtype="bf16", rows=4096, vocab=131072, ld=131072, mask=0, top=5),
        # a ragged batch: odd width, padded rows, constrained decoding masks, padding tokens,
        # rows that allow nothing
        dict(name="tokens_ragged", op="logprobs", dtype="f16", rows=777, vocab=50021, ld=50048, mask=1, top=8),
        # policy-gradient step over a stored rollout: values, then the gradient of the logits
        dict(name="actions_train", op="train", dtype="f32", rows=262144, vocab=43, ld=44, mask=0, top=0),
        # fine-tuning step of a language model
        dict(name="tokens_train", op="train", dtype="bf16", rows=2048, vocab=131072, ld=131072, mask=0, top=0),
        # the same with masks and with a loss on the alternatives too, odd sizes
        dict(name="tokens_train_odd", op="train", dtype="f16", rows=1001, vocab=32003, ld=32003, mask=1, top=8),
        # the nine gate blocks of three recurrent layers, 256 units: latency counts
        dict(name="gates", op="orthogonalize", dtype="f32", batch=9, rows=256, cols=256),
        # a large square weight in bf16
        dict(name="square_bf16", op="orthogonalize", dtype="bf16", batch=1, rows=4096, cols=4096),
        # the whole optimiser step of the encoder weight (843 features to 256 units)
        dict(name="encoder_step", op="muon", dtype="f32", batch=1, rows=843, cols=256),
        # the same for a feed-forward sized weight with odd sizes
        dict(name="wide_step", op="muon", dtype="f32", batch=1, rows=1000, cols=2731),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["logprobs", "train", "orthogonalize", "muon"])
    if op in ("logprobs", "train"):
        vocab = _log_int(rng, 2, 131072)
        most = 4096 * 131072 // (4 if op == "train" else 1)
        rows = _log_int(rng, 1, max(1, min(262144, most // 2 // vocab)))
        return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), rows=rows, vocab=vocab,
                    ld=vocab + rng.choice([0, 1, 5, 64]), mask=rng.choice([0, 0, 1]), top=rng.choice([0, 1, 5, 20, 32]))
    rows, cols = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
    small, large = min(rows, cols), max(rows, cols)
    most = 4 * 4096 ** 3 // 4 // (3 * small * small * large + small ** 3)
    return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]) if op == "orthogonalize" else "f32",
                batch=_log_int(rng, 1, max(1, min(16, most))), rows=rows, cols=cols)


def work(case):
    if case["op"] in ("logprobs", "train"):
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        elements = rows * vocab
        moved = elements * SIZES[case["dtype"]] + case["mask"] * elements + rows * (4 + 4 + 4 + 8 * top)
        if case["op"] == "train":
            moved += elements * SIZES[case["dtype"]] + rows * (4 + 4 + 4 * top)
        return {"bytes": moved, "flops": 0}
    # symmetric products need one half: X X^T m^2 n, A A m^3, B X 2 m^2 n
    small, large = min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    elements = case["batch"] * small * large
    moved = 2 * elements * SIZES[case["dtype"]] if case["op"] == "orthogonalize" else 5 * elements * 4
    return {"bytes": moved, "flops": case["batch"] * STEPS * (3 * small * small * large + small ** 3)}


# ---- inputs ------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    if case["op"] in ("logprobs", "train"):
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        store = normal(rows, case["ld"], dtype=DTYPES[case["dtype"]]).mul_(2.5)
        logits = store[:, :vocab]
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        at = torch.arange(rows, device="cuda")
        # a model that has learnt something: the given token stands out in three rows of four
        logits[at, tokens.long()] += torch.where(at % 4 == 0, 0.0, 6.0).to(logits.dtype)
        state = dict(case, logits=logits, mask=None)
        if case["mask"]:
            mask = (torch.rand(rows, vocab, generator=gen, device="cuda") < 0.8).to(torch.uint8)
            mask[at, tokens.long()] = 1
            mask[3::29] = 0            # rows that allow nothing
            state["mask"] = mask
            tokens[1::13] = -1         # padding
        state["tokens"] = tokens
        if case["op"] == "train":
            state["g_logprobs"] = normal(rows)      # advantages; 16-bit programs scale their loss
            state["g_entropy"] = normal(rows) * 0.01
            state["g_top"] = normal(rows, top) * 0.1 if top else None
        return state
    batch, rows, cols = case["batch"], case["rows"], case["cols"]
    # a gradient: sums of outer products whose weights fall off, so that the spectrum does
    rank = min(rows, cols)
    fall = torch.arange(1, rank + 1, device="cuda", dtype=torch.float32).rsqrt()
    grad = torch.matmul(normal(batch, rows, rank) * fall, normal(batch, rank, cols)) * 1e-3
    state = dict(case, grad=grad.to(DTYPES[case["dtype"]]))
    if case["op"] == "muon":
        state["weight"] = normal(batch, rows, cols) * cols ** -0.5
        state["momentum"] = normal(batch, rows, cols) * grad.std()
    return state


# ---- one pass ----------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "logprobs":
        d = _distribution(state)
        return _values(state, d)
    if op == "train":
        d = _distribution(state)
        out = _values(state, d)
        return dict(out, grad=_gradient(state, d, out))
    if op == "orthogonalize":
        return _orthogonal(state["grad"].float()).to(state["grad"].dtype)
    state["momentum"].mul_(MOMENTUM).add_(state["grad"])
    update = _orthogonal(state["grad"] + MOMENTUM * state["momentum"])
    scale = max(1.0, state["rows"] / state["cols"]) ** 0.5
    state["weight"].mul_(1.0 - LR * DECAY).sub_(LR * scale * update)
    return dict(weight=state["weight"], momentum=state["momentum"])


def _run_own(state):
    policy = _policy()
    op = state["op"]
    if op in ("logprobs", "train"):
        got = policy.token_logprobs(state["logits"], state["tokens"], mask=state["mask"], top=state["top"],
                                    stats=op == "train")
        out = dict(logprobs=got.logprobs, entropy=got.entropy)
        if state["top"]:
            out.update(top_ids=got.top_ids, top_logprobs=got.top_logprobs)
        if op == "train":
            out["grad"] = policy.token_logprobs_backward(
                state["logits"], state["tokens"], got.stats, g_logprobs=state["g_logprobs"],
                g_entropy=state["g_entropy"], mask=state["mask"], top_ids=got.top_ids, g_top=state["g_top"])
        return out
    if op == "orthogonalize":
        return policy.orthogonalize(state["grad"], steps=STEPS, eps=EPS)
    policy.muon_update(state["weight"], state["grad"], state["momentum"], LR, momentum=MOMENTUM,
                       weight_decay=DECAY, steps=STEPS, eps=EPS)
    return dict(weight=state["weight"], momentum=state["momentum"])


# ---- the plain forms ---------------------------------------------------------------------
def _distribution(state):
    """log p of every entry in 32 bits; -inf where the mask leaves nothing."""
    x = state["logits"].float()
    if state["mask"] is not None:
        x = x.masked_fill(state["mask"] == 0, -torch.inf)
    most = x.amax(1, keepdim=True)
    none = most == -torch.inf
    x = x - most.masked_fill(none, 0.0)
    p = x.exp()
    total = p.sum(1, keepdim=True)
    logp = x - total.log().masked_fill(none, 0.0)
    return logp, p / total.masked_fill(none, 1.0)


def _values(state, d):
    logp, p = d
    tokens = state["tokens"].long()
    taken = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    out = dict(logprobs=torch.where(tokens < 0, 0.0, taken), entropy=-(p * logp.clamp(min=-1e30)).sum(1))
    if state["top"]:
        out.update(zip(("top_ids", "top_logprobs"), _alternatives(state, logp)))
    return out


def _alternatives(state, logp):
    """The largest logits in order, ties to the lowest index: one 64-bit key an entry."""
    x = state["logits"].float() + 0.0
    vocab, top = state["vocab"], state["top"]
    bits = x.contiguous().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    key = order * vocab + torch.arange(vocab - 1, -1, -1, device=x.device)
    if state["mask"] is not None:
        key = key.masked_fill(state["mask"] == 0, torch.iinfo(torch.int64).min)
    best = key.topk(min(top, vocab), 1).values
    ids = vocab - 1 - torch.remainder(best, vocab)
    there = best != torch.iinfo(torch.int64).min
    shown = torch.where(there, logp.gather(1, torch.where(there, ids, 0)), -torch.inf)
    ids = torch.where(there, ids, -1).to(torch.int32)
    return (torch.nn.functional.pad(ids, (0, top - ids.shape[1]), value=-1),
            torch.nn.functional.pad(shown, (0, top - shown.shape[1]), value=-torch.inf))


def _gradient(state, d, values):
    """d(sum g lp + g_H H + sum g_top lp_top) / d logits, rounded once."""
    logp, p = d
    tokens = state["tokens"].long()
    entropy = values["entropy"][:, None]
    given = torch.where((tokens >= 0) & (logp.amax(1) > -torch.inf), state["g_logprobs"], 0.0)[:, None]
    weight = given.clone()
    out = torch.zeros_like(p)
    out.scatter_add_(1, tokens.clamp(min=0)[:, None], given)
    if state["g_top"] is not None:
        ids = values["top_ids"].long()
        g_top = torch.where(ids >= 0, state["g_top"], 0.0)
        out.scatter_add_(1, ids.clamp(min=0), g_top)
        weight = weight + g_top.sum(1, keepdim=True)
    out -= p * (weight + state["g_entropy"][:, None] * (logp.clamp(min=-1e30) + entropy))
    return out.to(state["logits"].dtype)


def _orthogonal(g):
    """STEPS quintic steps towards the nearest semi-orthogonal matrix, the norm in 64 bits."""
    a, b, c = QUINTIC
    tall = g.shape[1] > g.shape[2]
    x = g.transpose(1, 2) if tall else g
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt()
    x = (x / (norm + EPS)).float().contiguous()

    def step(x):
        s = torch.matmul(x, x.transpose(1, 2).contiguous())
        return a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)

    x = step(step(step(step(step(x)))))
    return x.transpose(1, 2).contiguous() if tall else x


# ---- the definitions in 64 bits ----------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("logprobs", "train"):
        return _exact_logprobs(case, s)
    grad = s["grad"].double()
    if case["op"] == "orthogonalize":
        return torch.stack([_exact_orthogonal(g) for g in grad])
    momentum = MOMENTUM * s["momentum"].double() + grad
    update = torch.stack([_exact_orthogonal(g) for g in grad + MOMENTUM * momentum])
    scale = max(1.0, case["rows"] / case["cols"]) ** 0.5
    weight = s["weight"].double()
    return dict(weight=weight - LR * (DECAY * weight + scale * update), momentum=momentum)


def _exact_orthogonal(g):
    """The polynomial written on the smaller Gram matrix' side, Horner's way."""
    a, b, c = QUINTIC
    x = g / (torch.linalg.vector_norm(g) + EPS)
    wide = x.shape[0] <= x.shape[1]
    eye = torch.eye(min(x.shape), dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        gram = x @ x.T.contiguous() if wide else x.T.contiguous() @ x
        p = a * eye + gram @ (b * eye + c * gram)
        x = p @ x if wide else x @ p
    return x


def _exact_logprobs(case, s):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    part = max(1, (1 << 27) // vocab)
    outs = []
    for r in range(0, rows, part):
        cut = slice(r, r + part)
        x = s["logits"][cut].double()
        allowed = torch.ones_like(x, dtype=torch.bool) if s["mask"] is None else s["mask"][cut] != 0
        tokens = s["tokens"][cut].long()
        some = allowed.any(1)
        x.requires_grad_(case["op"] == "train")
        # rows without any allowed entry go through the soft maximum unmasked and are set after it
        logp = torch.log_softmax(torch.where(allowed | ~some[:, None], x, -torch.inf), 1)
        given = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
        kept = logp.masked_fill(~(allowed & some[:, None]), 0.0)
        entropy = -(kept.exp() * kept).masked_fill(~(allowed & some[:, None]), 0.0).sum(1)
        empty = torch.full_like(given, -torch.inf)
        out = dict(logprobs=torch.where(tokens < 0, 0.0, torch.where(some, given, empty)).detach(),
                   entropy=entropy.detach())
        if top:
            shown = torch.sort(torch.where(allowed, s["logits"][cut].double(), -torch.inf), dim=1, descending=True,
                               stable=True)[1][:, :top]
            there = allowed.gather(1, shown)
            shown_lp = logp.gather(1, shown)
            out["top_logprobs"] = torch.nn.functional.pad(
                torch.where(there, shown_lp, -torch.inf), (0, top - shown.shape[1]), value=-torch.inf).detach()
            out["top_ids"] = None
        if case["op"] == "train":
            loss = (torch.where((tokens >= 0) & some, given, 0.0) * s["g_logprobs"][cut].double()).sum()
            loss = loss + (entropy * s["g_entropy"][cut].double()).sum()
            if top:
                g_top = s["g_top"][cut].double()[:, :shown.shape[1]]
                loss = loss + (torch.where(there, shown_lp, 0.0) * g_top).sum()
            out["grad"] = torch.autograd.grad(loss, x)[0]
        outs.append(out)
    return {k: None if outs[0][k] is None else torch.cat([o[k] for o in outs]) for k in outs[0]}
