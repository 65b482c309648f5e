"""Training by preference and by reward, as cases that can be timed and compared: dropout between
layers, the log-probability of the chosen class or token, the clipped policy loss with a KL term
and the preference loss of paired sequences, each with its gradient.

Each case is a dict of plain values.  `listed` gives the named ones, `draw` one more of the same
ranges; `prepare` makes what a program holds before the call, `run` makes one pass (the plain
formulas in torch, or the framework's operators where `own` is true), `exact` restates the pass
in 64 bits from the definitions, `work` counts what the pass cannot do without.

Kinds:
  dropout     a forward and a backward pass over activations [rows, cols]; layout "rows"
              (cols contiguous) or "columns" (the view of [cols, rows] that a LogicLayer gives);
              fill "scale" (dropped 0, kept divided by the keep probability) or a constant
              (dropped become it, kept stay as they are)
  log_probs   the log-probability of one class or token per row, and the logits' gradient
  policy      the clipped policy loss with a KL term, and the logits' gradient
  group       the same through GroupSum: class scores from a network's last activations, and the
              gradient of those
  preference  the preference loss of paired ragged sequences, and the logits' gradient
"""
import numpy as np
import torch

own = False

CLASSES = 10
IGNORE = -100
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
KL = 0.05
BETA = 0.1
SMOOTHING = 0.02
LARGEST = 8192 * 32768          # logits of the largest listed case
LARGEST_DROPOUT = 16384 * 11999


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the input of a first experiment: 100 samples of 28 x 28 bits, where a call's latency counts
        _dropout("dropout_small", 100, 784, "rows", "float32", 0.1, "scale"),
        # a hidden LogicLayer's relaxed activations, unknown bits instead of zeros
        _dropout("dropout_layer", 1024, 12000, "columns", "float32", 0.05, 0.5),
        # wide half-width activations whose rows end anywhere
        _dropout("dropout_ragged", 16384, 11999, "rows", "bfloat16", 0.25, "scale"),
        # scores of a 200-class network for a batch of samples
        _tokens("log_probs_scores", "log_probs", 1024, 200, "float32", 0),
        # a vocabulary that no tile divides, a fifth of the rows padding
        _tokens("log_probs_vocab", "log_probs", 4096, 50021, "bfloat16", 20),
        # a policy over ten actions: the smallest step
        _tokens("policy_small", "policy", 128, 10, "float32", 0),
        # the same from a logic network's last activations
        _group("policy_group", 1024, 12000),
        # a batch of sampled answers, prompts and padding ignored
        _tokens("policy_tokens", "policy", 8192, 32768, "bfloat16", 25),
        # odd rows and an odd vocabulary in full precision
        _tokens("policy_ragged", "policy", 2047, 32003, "float32", 10),
        # few rows with a long vocabulary: the last tokens of a few answers
        _tokens("policy_long", "policy", 16, 131072, "float16", 0),
        # pairs of single answers of a 200-class network
        _preference("preference_scores", 64, 1, 200, "float32"),
        # pairs of ragged answers
        _preference("preference_tokens", 16, 256, 32000, "bfloat16"),
    ]


def draw(rng):
    def size(lo, hi):
        """Log-uniform in [lo, hi]."""
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["dropout", "dropout", "dropout", "log_probs", "log_probs", "policy", "policy",
                       "policy", "group", "preference", "preference"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind == "dropout":
        cols = size(64, 16384)
        rows = min(size(16, 16384), LARGEST_DROPOUT // cols)
        case = _dropout("", rows, cols, rng.choice(["rows", "columns"]), dtype,
                        round(rng.uniform(0.02, 0.6), 3), rng.choice(["scale", 0.5]))
    elif kind == "group":
        case = _group("", size(32, 1024), size(500, 12000))
    else:
        limit = LARGEST if dtype != "float32" else LARGEST // 2
        vocab = size(5, 131072)
        if kind == "preference":
            pairs = size(2, 64)
            most = max(1, limit // (4 * vocab * pairs))
            case = _preference("", pairs, min(size(1, 512), most), vocab, dtype)
        else:
            rows = min(size(16, 16384), limit // vocab)
            case = _tokens("", kind, rows, vocab, dtype, rng.choice([0, 0, 10, 30]))
    case.pop("name", None)
    return case


def _dropout(name, rows, cols, layout, dtype, p, fill):
    return {"name": name, "kind": "dropout", "rows": rows, "cols": cols, "layout": layout,
            "dtype": dtype, "p": p, "fill": fill}


def _tokens(name, kind, rows, vocab, dtype, ignored_percent):
    return {"name": name, "kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype,
            "ignored": rows * ignored_percent // 100}


def _group(name, batch, features):
    return {"name": name, "kind": "group", "rows": batch, "features": features}


def _preference(name, pairs, length, vocab, dtype):
    return {"name": name, "kind": "preference", "pairs": pairs, "length": length, "vocab": vocab,
            "dtype": dtype, "rows": 2 * pairs * length}


# ------------------------------------------------------------------------------------ prepare

def prepare(case, seed):
    return {"dropout": _prepare_dropout, "group": _prepare_group, "preference": _prepare_preference,
            "log_probs": _prepare_tokens, "policy": _prepare_tokens}[case["kind"]](case, seed)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_dropout(case, seed):
    """Relaxed activations in [0, 1], the gradient of a mean loss, and the generator's state."""
    gen = _generator(seed)
    shape = (case["rows"], case["cols"])
    lies = shape if case["layout"] == "rows" else shape[::-1]
    dtype = getattr(torch, case["dtype"])
    x = torch.rand(lies, generator=gen, device="cuda").to(dtype)
    gy = torch.randn(lies, generator=gen, device="cuda").to(dtype)
    if case["layout"] != "rows":
        x, gy = x.t(), gy.t()
    rng = torch.randint(0, 1 << 62, (2,), generator=gen, device="cuda")
    return {"kind": "dropout", "case": case, "x": x.requires_grad_(), "gy": gy, "rng": rng}


def _choose(logits, gen):
    """One action per row, drawn from the softmax of the logits, and its log-probability."""
    z = logits.float()
    noise = torch.empty_like(z).exponential_(generator=gen).log_()
    actions = (z - noise).argmax(1)
    lp = torch.gather(z, 1, actions[:, None])[:, 0] - torch.logsumexp(z, 1)
    return actions, lp


def _logits(rows, vocab, dtype, gen):
    return (torch.randn((rows, vocab), generator=gen, device="cuda") * 2.5).to(dtype)


def _prepare_tokens(case, seed):
    """Logits, the tokens chosen, and what the acting and the reference policy gave them."""
    gen = _generator(seed)
    rows = case["rows"]
    logits = _logits(rows, case["vocab"], getattr(torch, case["dtype"]), gen)
    actions, lp = _choose(logits, gen)
    old = lp + 0.15 * torch.randn(rows, generator=gen, device="cuda")
    ref = lp + 0.3 * torch.randn(rows, generator=gen, device="cuda")
    adv = torch.randn(rows, generator=gen, device="cuda")
    where = torch.rand(rows, generator=gen, device="cuda").argsort()[:case["ignored"]]
    actions[where] = IGNORE
    return {"kind": case["kind"], "case": case, "logits": logits.requires_grad_(),
            "actions": actions, "old": old, "ref": ref, "adv": adv}


def _prepare_group(case, seed):
    """Activations of a network's last layer as it hands them on, ten actions."""
    gen = _generator(seed)
    x = torch.rand((case["features"], case["rows"]), generator=gen, device="cuda").t()
    size = -(-case["features"] // CLASSES)
    padded = torch.nn.functional.pad(x, (0, size * CLASSES - case["features"]))
    tau = float(max(1.0, size ** 0.5 / 8))
    scores = padded.reshape(case["rows"], CLASSES, size).sum(2) / tau
    actions, lp = _choose(scores, gen)
    rows = case["rows"]
    old = lp + 0.15 * torch.randn(rows, generator=gen, device="cuda")
    ref = lp + 0.3 * torch.randn(rows, generator=gen, device="cuda")
    adv = torch.randn(rows, generator=gen, device="cuda")
    return {"kind": "group", "case": case, "x": x.requires_grad_(), "actions": actions, "old": old,
            "ref": ref, "adv": adv, "tau": tau, "size": size}


def _prepare_preference(case, seed):
    """Chosen sequences, then rejected ones, in one ragged batch of tokens, each at least one
    token long; the reference's log-probabilities."""
    gen = _generator(seed)
    count, rows = 2 * case["pairs"], case["rows"]
    inner = torch.randperm(rows - 1, generator=gen, device="cuda")[:count - 1].sort().values + 1
    even = torch.arange(1, count, device="cuda") * case["length"]
    cuts = (inner + even + 1) // 2 if case["length"] > 1 else even
    offsets = torch.cat((cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)))
    logits = _logits(rows, case["vocab"], getattr(torch, case["dtype"]), gen)
    actions, lp = _choose(logits, gen)
    ref = lp + 0.2 * torch.randn(rows, generator=gen, device="cuda")
    return {"kind": "preference", "case": case, "logits": logits.requires_grad_(),
            "actions": actions, "ref": ref, "offsets": offsets}


# ------------------------------------------------------------------------------------ run

def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _own_dropout(state):
    import compactlogic_amd as cl
    case = state["case"]
    fill = None if case["fill"] == "scale" else case["fill"]
    y = cl.dropout(state["x"], case["p"], state["rng"], fill=fill)
    (gx,) = torch.autograd.grad(y, state["x"], state["gy"])
    return {"y": y.detach(), "grad": gx}


def _own_log_probs(state):
    import compactlogic_amd as cl
    lp = cl.selected_log_probs(state["logits"], state["actions"])
    (grad,) = torch.autograd.grad(lp, state["logits"], state["adv"])
    return {"log_probs": lp.detach(), "grad": grad}


def _own_policy(state):
    import compactlogic_amd as cl
    loss, lp = cl.policy_loss(state["logits"], state["actions"], state["old"], state["adv"],
                              ref_log_probs=state["ref"], clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL,
                              return_log_probs=True)
    (grad,) = torch.autograd.grad(loss, state["logits"])
    return {"loss": loss.detach(), "log_probs": lp, "grad": grad}


def _own_group(state):
    import compactlogic_amd as cl
    loss, lp = cl.GroupSum(CLASSES, state["tau"]).policy_loss(
        state["x"], state["actions"], state["old"], state["adv"], ref_log_probs=state["ref"],
        clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL, return_log_probs=True)
    (grad,) = torch.autograd.grad(loss, state["x"])
    return {"loss": loss.detach(), "log_probs": lp, "grad": grad}


def _own_preference(state):
    import compactlogic_amd as cl
    loss, margins = cl.preference_loss(state["logits"], state["actions"], state["offsets"],
                                       ref_log_probs=state["ref"], beta=BETA,
                                       label_smoothing=SMOOTHING, return_margins=True)
    (grad,) = torch.autograd.grad(loss, state["logits"])
    return {"loss": loss.detach(), "margins": margins, "grad": grad}


def _philox(c0, c1, c2, c3, k0, k1):
    """Ten rounds of Philox 4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
    as 1, 2, 3", 2011) on int64 tensors that hold 32-bit words."""
    word = 0xFFFFFFFF
    for _ in range(10):
        lo0, lo2 = 0xD2511F53 * (c0 & 0xFFFF), 0xCD9E8D57 * (c2 & 0xFFFF)
        hi0, hi2 = 0xD2511F53 * (c0 >> 16) + (lo0 >> 16), 0xCD9E8D57 * (c2 >> 16) + (lo2 >> 16)
        c0, c1, c2, c3 = ((hi2 >> 16) ^ c1 ^ k0,
                          ((hi2 & 0xFFFF) << 16) | (lo2 & 0xFFFF),
                          (hi0 >> 16) ^ c3 ^ k1,
                          ((hi0 & 0xFFFF) << 16) | (lo0 & 0xFFFF))
        k0, k1 = (k0 + 0x9E3779B9) & word, (k1 + 0xBB67AE85) & word
    return c0, c1, c2, c3


def _threshold(p):
    return int(round(65536 * p))


def _plain_dropout(state):
    case, rng = state["case"], state["rng"]
    x, gy = state["x"].detach(), state["gy"]
    rows, cols = x.shape
    t = _threshold(case["p"])
    block = torch.arange(-(-cols // 8), device=x.device).expand(rows, -1)
    row = torch.arange(rows, device=x.device)[:, None].expand_as(block)
    seed, offset = rng[0], rng[1]
    words = _philox(block, row, offset & 0xFFFFFFFF, (offset >> 32) & 0xFFFFFFFF,
                    seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 2)
    keep = halves.reshape(rows, -1)[:, :cols] >= t
    if case["fill"] == "scale":
        scale, fill = 65536.0 / (65536 - t), 0.0
    else:
        scale, fill = 1.0, case["fill"]
    y = torch.where(keep, x.float() * scale, fill).to(x.dtype)
    gx = torch.where(keep, gy.float() * scale, 0.0).to(x.dtype)
    return {"y": y, "grad": gx}


def _log_softmax_parts(x, actions):
    """(chosen, counted rows, their log-probability in 64 bits, probabilities) of logits x."""
    counted = actions != IGNORE
    chosen = torch.where(counted, actions, 0)
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    lp = torch.gather(x, 1, chosen[:, None]).double() - m.double() - torch.log(s.double())
    return chosen, counted, lp[:, 0], e / s


def _logit_gradient(probs, chosen, row_gradient):
    """row_gradient * (1[j = chosen] - probs)."""
    grad = probs * -row_gradient[:, None]
    return grad.scatter_add_(1, chosen[:, None], row_gradient[:, None])


def _plain_log_probs(state):
    x = state["logits"].detach()
    chosen, counted, lp, probs = _log_softmax_parts(x.float(), state["actions"])
    g = torch.where(counted, state["adv"], 0.0)
    return {"log_probs": torch.where(counted, lp, 0.0).float(),
            "grad": _logit_gradient(probs, chosen, g).to(x.dtype)}


def _policy_terms(lp, counted, state):
    """The loss, and its derivative by each row's log-probability, in 64 bits: rows lie next to
    the borders of the clipped range."""
    old, ref, adv = state["old"].double(), state["ref"].double(), state["adv"].double()
    ratio = torch.exp(lp - old)
    free, bound = ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    far = torch.exp(ref - lp)
    term = KL * (far - (ref - lp) - 1) - torch.minimum(free, bound)
    slope = KL * (1 - far) - torch.where(free <= bound, free, 0.0)
    count = counted.sum()
    return (torch.where(counted, term, 0.0).sum() / count,
            torch.where(counted, slope, 0.0) / count)


def _plain_policy(state):
    x = state["logits"].detach()
    chosen, counted, lp, probs = _log_softmax_parts(x.float(), state["actions"])
    loss, slope = _policy_terms(lp, counted, state)
    return {"loss": loss.float(), "log_probs": torch.where(counted, lp, 0.0).float(),
            "grad": _logit_gradient(probs, chosen, slope.float()).to(x.dtype)}


def _plain_group(state):
    x = state["x"].detach()
    rows, features = x.shape
    size = state["size"]
    padded = torch.zeros((rows, size * CLASSES), device=x.device)
    padded[:, :features] = x
    scores = padded.reshape(rows, CLASSES, size).sum(2) / state["tau"]
    chosen, counted, lp, probs = _log_softmax_parts(scores, state["actions"])
    loss, slope = _policy_terms(lp, counted, state)
    grad = _logit_gradient(probs, chosen, slope.float()) / state["tau"]
    group = torch.arange(features, device=x.device) // size
    return {"loss": loss.float(), "log_probs": lp.float(), "grad": grad.t()[group].t()}


def _plain_preference(state):
    x, offsets = state["logits"].detach(), state["offsets"]
    pairs = state["case"]["pairs"]
    chosen, counted, lp, probs = _log_softmax_parts(x.float(), state["actions"])
    parts = torch.where(counted, lp - state["ref"].double(), 0.0)
    sums = torch.cat((parts.new_zeros(1), torch.cumsum(parts, 0)))
    ratio = sums[offsets[1:]] - sums[offsets[:-1]]
    h = BETA * (ratio[:pairs] - ratio[pairs:])
    away, near = torch.log1p(torch.exp(-h.abs())) - h.clamp(max=0), \
        torch.log1p(torch.exp(-h.abs())) + h.clamp(min=0)
    loss = ((1 - SMOOTHING) * away + SMOOTHING * near).mean()
    slope = BETA / pairs * (SMOOTHING / (1 + torch.exp(-h)) - (1 - SMOOTHING) / (1 + torch.exp(h)))
    row = torch.arange(x.shape[0], device=x.device)
    sequence = (row[:, None] >= offsets[None, 1:]).sum(1)
    g = torch.where(counted, torch.cat((slope, -slope))[sequence], 0.0)
    return {"loss": loss.float(), "margins": h.float(),
            "grad": _logit_gradient(probs, chosen, g.float()).to(x.dtype)}


_PLAIN = {"dropout": _plain_dropout, "log_probs": _plain_log_probs, "policy": _plain_policy,
          "group": _plain_group, "preference": _plain_preference}
_OWN = {"dropout": _own_dropout, "log_probs": _own_log_probs, "policy": _own_policy,
        "group": _own_group, "preference": _own_preference}


# ------------------------------------------------------------------------------------ work

def work(case):
    """Bytes: inputs read once, outputs written once.  Operations per logit: a difference, an
    exponential and a sum for the softmax, two products for the gradient; per dropped or kept
    element a comparison and a product each way and its eighth of ten generator rounds (two
    products, four exclusive ors) each way."""
    size = {"float32": 4, "float16": 2, "bfloat16": 2}.get(case.get("dtype"), 4)
    rows = case["rows"]
    if case["kind"] == "dropout":
        n = rows * case["cols"]
        return {"bytes": 4 * n * size, "flops": n * (4 + 2 * 60 // 8)}
    if case["kind"] == "group":
        n = rows * case["features"]
        return {"bytes": 8 * n + 24 * rows, "flops": 2 * n + 50 * rows}
    vocab = case["vocab"]
    read = rows - case.get("ignored", 0)
    per_row = {"log_probs": 16, "policy": 24, "preference": 12}[case["kind"]]
    return {"bytes": (read + rows) * vocab * size + per_row * rows, "flops": 5 * read * vocab}


# ------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return {"dropout": _exact_dropout, "log_probs": _exact_tokens, "policy": _exact_tokens,
            "group": _exact_group, "preference": _exact_preference}[case["kind"]](case, state)


def _exact_keep(case, seed, offset):
    """The mask from the generator's definition, in unsigned host arithmetic, a band of rows at a
    time."""
    rows, cols = case["rows"], case["cols"]
    blocks = -(-cols // 8)
    low = np.uint64(0xFFFFFFFF)
    t = _threshold(case["p"])
    keep = np.empty((rows, cols), dtype=bool)
    band = max(1, 65536 // blocks)
    for r0 in range(0, rows, band):
        r = np.arange(r0, min(rows, r0 + band), dtype=np.uint64)
        ctr = [np.tile(np.arange(blocks, dtype=np.uint64), len(r)), np.repeat(r, blocks),
               np.uint64(offset & 0xFFFFFFFF), np.uint64(offset >> 32)]
        for i in range(10):
            ka = np.uint64(((seed & 0xFFFFFFFF) + i * 0x9E3779B9) & 0xFFFFFFFF)
            kb = np.uint64(((seed >> 32) + i * 0xBB67AE85) & 0xFFFFFFFF)
            a, b = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
            ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ ka, b & low, (a >> np.uint64(32)) ^ ctr[3] ^ kb, a & low]
        quad = np.stack([np.broadcast_to(c, (len(r) * blocks,)) for c in ctr], 1).astype("<u4")
        keep[r0:r0 + len(r)] = quad.view("<u2").reshape(len(r), blocks * 8)[:, :cols] >= t
    return keep


def _exact_dropout(case, state):
    seed, offset = (int(v) for v in state["rng"].tolist())
    keep = torch.from_numpy(_exact_keep(case, seed, offset)).cuda()
    x, gy = state["x"].detach().double(), state["gy"].double()
    if case["fill"] == "scale":
        rate = 1.0 - _threshold(case["p"]) / 65536.0
        return {"y": (x / rate).masked_fill_(~keep, 0.0), "grad": (gy / rate).masked_fill_(~keep, 0.0)}
    return {"y": x.masked_fill(~keep, case["fill"]), "grad": gy.masked_fill(~keep, 0.0)}


def _exact_row_log_probs(z, actions):
    """Log-probability of each counted row's action (0 elsewhere) of 64-bit logits z."""
    counted = actions != IGNORE
    rows = torch.arange(z.shape[0], device=z.device)[counted]
    lp = torch.log_softmax(z, 1)
    return z.new_zeros(z.shape[0]).index_put((rows,), lp[rows, actions[counted]]), counted


def _exact_policy_loss(lp, counted, state):
    old, ref, adv = (state[k].double()[counted] for k in ("old", "ref", "adv"))
    own_lp = lp[counted]
    ratio = torch.exp(own_lp - old)
    gain = torch.where(adv >= 0, torch.clamp(ratio, max=1 + CLIP_HIGH),
                       torch.clamp(ratio, min=1 - CLIP_LOW)) * adv
    gap = ref - own_lp
    return (KL * (torch.expm1(gap) - gap) - gain).mean()


def _exact_tokens(case, state):
    z = state["logits"].detach().double().requires_grad_()
    lp, counted = _exact_row_log_probs(z, state["actions"])
    if case["kind"] == "log_probs":
        (grad,) = torch.autograd.grad(lp, z, state["adv"].double())
        return {"log_probs": lp.detach(), "grad": grad}
    loss = _exact_policy_loss(lp, counted, state)
    (grad,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "log_probs": lp.detach(), "grad": grad}


def _exact_group(case, state):
    x = state["x"].detach().double().requires_grad_()
    scores = torch.stack([part.sum(1) for part in _groups(x, state["size"])], 1) / state["tau"]
    lp, counted = _exact_row_log_probs(scores, state["actions"])
    loss = _exact_policy_loss(lp, counted, state)
    (grad,) = torch.autograd.grad(loss, x)
    return {"loss": loss.detach(), "log_probs": lp.detach(), "grad": grad}


def _groups(x, size):
    """The features of each class; the last classes may have fewer, or none."""
    return [x[:, c * size:(c + 1) * size] for c in range(CLASSES)]


def _exact_preference(case, state):
    z = state["logits"].detach().double().requires_grad_()
    lp, _ = _exact_row_log_probs(z, state["actions"])
    gap = lp - state["ref"].double()
    ends = state["offsets"].tolist()
    ratio = torch.stack([gap[a:b].sum() for a, b in zip(ends[:-1], ends[1:])])
    h = BETA * (ratio[:case["pairs"]] - ratio[case["pairs"]:])
    logsigmoid = torch.nn.functional.logsigmoid
    loss = -((1 - SMOOTHING) * logsigmoid(h) + SMOOTHING * logsigmoid(-h)).mean()
    (grad,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "margins": h.detach(), "grad": grad}
