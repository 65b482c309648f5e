"""Sequences of logic activations, the step that trains on them and the answers drawn from them, as
cases that can be timed and compared.

Each case is a dict of plain values.  `listed` gives the named ones, `draw` one more of the same
ranges; `prepare` makes what a program holds before the call, `run` makes one pass (the plain
formulas in torch, or the framework's operators where `own` is true), `exact` restates the pass
in 64 bits from the definitions, `work` counts what the pass cannot do without.

Kinds:
  adamw       one step over many tensors with the gradient's norm clipped, moments in 32 bits or
              in 8 (blocks of 256: exp_avg in e4m3, exp_avg_sq in an unsigned type of five
              exponent and three mantissa bits, each with a power of two per block); returns the
              parameters and the moments
  recurrence  a gated linear recurrence over x, gate [batch, time, features], form "mix"
              (h = g h + (1 - g) x) or "add" (h = g h + x), lying with its features contiguous
              ("rows") or its times ("columns": what a LogicLayer gives for batch * time samples);
              "train": outputs, last state and all gradients, else outputs and last state
  verify      drafted tokens against the target's probabilities: how many are accepted, the tokens
              that result, the target's log-probabilities of them
"""
import torch

own = False

IGNORE = -100
BLOCK = 256                       # elements that share a power of two
LR, BETAS, EPS, MAX_NORM = 0.002, (0.9, 0.98), 1e-8, 1.0
STEPS_BEFORE = 100
LARGEST_ADAMW = 37_000_000        # elements in half width with small moments; else half as many
LARGEST_RECURRENCE = 8 * 4096 * 2048
LARGEST_VERIFY = 64 * 11 * 50021  # target's and draft's logits


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # a first experiment's two small layers, where a call's latency counts
        _adamw("adamw_small", 2, 1536, "float32", 32),
        # six layers of 12000 neurons with 16 gates each
        _adamw("adamw_network", 6, 192000, "float32", 32),
        # hundreds of tensors of any size in half width, most of them small
        _adamw("adamw_many", 192, 1_000_003, "bfloat16", 32),
        # a few long tensors in full precision with small moments
        _adamw("adamw8_network", 6, 256000, "float32", 8),
        # the most elements: half width, small moments
        _adamw("adamw8_large", 12, 20_000_003, "bfloat16", 8),
        # one new step of 64 sequences, a network of 12000 features: latency
        _recurrence("recurrence_token", 64, 1, 12000, "columns", "float32", "mix", False),
        # training on short sequences as LogicLayers hand them on
        _recurrence("recurrence_columns", 64, 64, 12000, "columns", "float32", "mix", True),
        # long sequences of wide half-width features
        _recurrence("recurrence_rows", 8, 4096, 2048, "rows", "bfloat16", "add", True),
        # one very long sequence of few features, odd in every size
        _recurrence("recurrence_long", 1, 65521, 251, "rows", "float32", "mix", True),
        # four drafted actions of ten for each of 256 episodes
        _verify("verify_scores", 256, 4, 10, "float32", 20),
        # one answer with a long vocabulary
        _verify("verify_one", 1, 7, 131072, "float32", 0),
        # a batch of answers, a vocabulary that no tile divides, some drafts shorter
        _verify("verify_tokens", 64, 5, 50021, "bfloat16", 20),
    ]


def draw(rng):
    def size(lo, hi):
        """Log-uniform in [lo, hi]."""
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["adamw", "adamw", "recurrence", "recurrence", "recurrence", "verify", "verify"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind == "adamw":
        bits = rng.choice([32, 8])
        count = size(1, 192 if bits == 32 else 20)
        case = _adamw("", count, size(100, 20_000_000), dtype, bits)
        total = sum(_sizes(case))
        most = LARGEST_ADAMW // (2 if dtype == "float32" or bits == 32 else 1)
        case["largest"] = case["largest"] * min(total, most) // total
    elif kind == "recurrence":
        train = rng.random() < 0.7
        time = size(2, 65536) if train else rng.choice([1, 1, size(2, 4096)])
        batch = size(1, 256)
        features = size(16, 16384)
        limit = LARGEST_RECURRENCE // (1 if dtype != "float32" else 2)
        batch = max(1, min(batch, limit // (time * features)))
        features = max(16, min(features, limit // (time * batch)))
        case = _recurrence("", batch, time, features, rng.choice(["rows", "columns"]), dtype,
                           rng.choice(["mix", "add"]), train)
    else:
        vocab, drafts = size(5, 131072), rng.randint(1, 8)
        limit = LARGEST_VERIFY // (1 if dtype != "float32" else 2)
        case = _verify("", min(size(1, 256), max(1, limit // ((2 * drafts + 1) * vocab))), drafts,
                       vocab, dtype, rng.choice([0, 0, 20]))
    case.pop("name", None)
    return case


def _adamw(name, tensors, largest, dtype, bits):
    return {"name": name, "kind": "adamw", "tensors": tensors, "largest": largest, "dtype": dtype,
            "bits": bits}


def _recurrence(name, batch, time, features, layout, dtype, form, train):
    return {"name": name, "kind": "recurrence", "batch": batch, "time": time, "features": features,
            "layout": layout, "dtype": dtype, "form": form, "train": train}


def _verify(name, sequences, drafts, vocab, dtype, short_percent):
    return {"name": name, "kind": "verify", "sequences": sequences, "drafts": drafts,
            "vocab": vocab, "dtype": dtype, "short": sequences * short_percent // 100}


def _sizes(case):
    """Elements of each tensor: equal layers where they are few, else sizes falling from the
    largest to a few elements, odd ones among them."""
    n, most = case["tensors"], case["largest"]
    if n <= 6:
        return [max(1, most - i * (most // 16)) for i in range(n)]
    return [max(1, int(most * (1.0 - i / n) ** 8)) for i in range(n)]


# ------------------------------------------------------------------------------------ prepare

def prepare(case, seed):
    return {"adamw": _prepare_adamw, "recurrence": _prepare_recurrence,
            "verify": _prepare_verify}[case["kind"]](case, seed)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_adamw(case, seed):
    """Parameters, gradients and moments of a run under way, each kind in one buffer of which the
    tensors are parts; every other tensor is decayed."""
    gen = _generator(seed)
    dtype = getattr(torch, case["dtype"])
    sizes = _sizes(case)
    total = sum(sizes)
    flat = torch.randn(total, generator=gen, device="cuda").to(dtype)
    grad = torch.randn(total, generator=gen, device="cuda")
    grad = (grad * grad.abs() * 0.02).to(dtype)
    first = torch.randn(total, generator=gen, device="cuda") * 0.01
    second = torch.rand(total, generator=gen, device="cuda").square_() * 4e-4 + first * first
    if case["bits"] == 8:
        first = torch.cat([_held_first(m) for m in first.split(sizes)])
        second = torch.cat([_held_second(v) for v in second.split(sizes)])
    params = [torch.nn.Parameter(p) for p in flat.split(sizes)]
    for p, g in zip(params, grad.split(sizes)):
        p.grad = g
    return {"kind": "adamw", "case": case, "flat": flat, "grad": grad, "params": params,
            "first": first, "second": second, "sizes": sizes, "steps": STEPS_BEFORE}


def _lies(t, layout):
    """t [batch, time, features] with its values, lying as `layout` says."""
    if layout == "rows":
        return t.contiguous()
    return t.permute(2, 0, 1).contiguous().permute(1, 2, 0)


def _prepare_recurrence(case, seed):
    """Relaxed activations, gates near and at their ends among them, a state carried over, and
    the gradients of what comes out."""
    gen = _generator(seed)
    dtype, layout = getattr(torch, case["dtype"]), case["layout"]
    shape = (case["batch"], case["time"], case["features"])
    gate = torch.randn(shape, generator=gen, device="cuda").mul_(1.5).add_(1.0).sigmoid_()
    if case["form"] == "mix":
        ends = torch.rand(shape, generator=gen, device="cuda")
        gate.masked_fill_(ends < 0.02, 0.0).masked_fill_(ends > 0.97, 1.0)
        x = torch.rand(shape, generator=gen, device="cuda")
    else:
        x = torch.randn(shape, generator=gen, device="cuda")
    state = torch.rand((shape[0], shape[2]), generator=gen, device="cuda")
    gy = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    gs = torch.randn((shape[0], shape[2]), generator=gen, device="cuda")
    x, gate, gy = (_lies(t.to(dtype), layout) for t in (x, gate, gy))
    if case["train"]:
        x, gate, state = x.requires_grad_(), gate.requires_grad_(), state.requires_grad_()
    return {"kind": "recurrence", "case": case, "x": x, "gate": gate, "state": state, "gy": gy,
            "gs": gs}


def _prepare_verify(case, seed):
    """The target's logits behind each drafted token and behind the last, the draft's logits and
    the tokens it drew from them, and the random numbers."""
    gen = _generator(seed)
    s, k, v = case["sequences"], case["drafts"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    logits = (torch.randn((s, k + 1, v), generator=gen, device="cuda") * 2.5).to(dtype)
    noise = torch.randn((s, k, v), generator=gen, device="cuda") * 0.5
    draft = (logits[:, :k].float() + noise).to(dtype)
    z = draft.float()
    tokens = (z - torch.empty_like(z).exponential_(generator=gen).log_()).argmax(2)
    where = torch.rand(s, generator=gen, device="cuda").argsort()[:case["short"]]
    lengths = torch.full((s,), k, device="cuda")
    lengths[where] = torch.randint(0, k, (case["short"],), generator=gen, device="cuda")
    tokens.masked_fill_(torch.arange(k, device="cuda") >= lengths[:, None], IGNORE)
    uniforms = torch.rand((s, k + 1), generator=gen, device="cuda")
    return {"kind": "verify", "case": case, "logits": logits, "draft": draft, "tokens": tokens,
            "uniforms": uniforms}


# ------------------------------------------------------------------------------------ run

def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _optimizer(state):
    """The program's optimizer, resumed from the moments of its checkpoint."""
    import compactlogic_amd as cl
    case, params = state["case"], state["params"]
    opt = cl.FusedAdamW([{"params": params[::2], "weight_decay": 0.1},
                         {"params": params[1::2], "weight_decay": 0.0}],
                        lr=LR, betas=BETAS, eps=EPS, max_norm=MAX_NORM, state_bits=case["bits"])
    first, second = state["first"].split(state["sizes"]), state["second"].split(state["sizes"])
    order = [*range(0, len(params), 2), *range(1, len(params), 2)]
    held = {i: {"step": torch.tensor(float(state["steps"])), "exp_avg": first[j],
                "exp_avg_sq": second[j]} for i, j in enumerate(order)}
    opt.load_state_dict({"state": held, "param_groups": opt.state_dict()["param_groups"]})
    return opt


def _own_adamw(state):
    opt = state.get("optimizer")
    if opt is None:
        opt = state["optimizer"] = _optimizer(state)
    opt.step()
    if state["case"]["bits"] == 32:
        return {"params": state["flat"], "first": state["first"], "second": state["second"]}
    first, second = opt.moments(state["params"])
    return {"params": state["flat"], "first": first, "second": second}


def _own_recurrence(state):
    import compactlogic_amd as cl
    x, gate, h0 = state["x"], state["gate"], state["state"]
    y, last = cl.gated_recurrence(x, gate, h0, form=state["case"]["form"], return_state=True)
    out = {"y": y.detach(), "last": last.detach()}
    if state["case"]["train"]:
        grads = torch.autograd.grad((y, last), (x, gate, h0), (state["gy"], state["gs"]))
        out.update(zip(("grad_x", "grad_gate", "grad_state"), grads))
    return out


def _own_verify(state):
    import compactlogic_amd as cl
    tokens, accepted, log_probs = cl.verify_drafts(state["logits"], state["tokens"], state["draft"],
                                                   state["uniforms"])
    return {"tokens": tokens, "accepted": accepted, "log_probs": log_probs}


def _blocks(t):
    """t in rows of one block each, the last one filled up with zeros."""
    n = t.numel()
    return torch.nn.functional.pad(t.reshape(-1), (0, -n % BLOCK)).reshape(-1, BLOCK)


def _power(blocks):
    """The exponent of each block's largest magnitude, at least -126."""
    return torch.frexp(blocks.abs().amax(1, keepdim=True)).exponent.sub(1).clamp(min=-126)


def _held_first(m):
    """m as e4m3 holds it, each block's largest magnitude in [128, 256) times a power of two."""
    b = _blocks(m)
    k = (_power(b) - 7).clamp(min=-126)
    codes = torch.ldexp(b, -k).to(torch.float8_e4m3fn)
    return torch.ldexp(codes.float(), k).reshape(-1)[:m.numel()]


def _held_second(v):
    """v >= 0 as five bits of exponent and three of mantissa hold it, each block's largest in
    [1, 2) times a power of two; what is not 0 stays at least the smallest code."""
    b = _blocks(v)
    k = _power(b)
    u = torch.ldexp(b, -k)
    bits = u.view(torch.int32)
    code = (bits + 0x7FFFF + ((bits >> 20) & 1) >> 20) - 770
    code = torch.where(u > 0, code.clamp(min=1), 0)
    held = torch.where(code > 0, ((code + 770) << 20).view(torch.float32), 0.0)
    return torch.ldexp(held, k).reshape(-1)[:v.numel()]


def _plain_adamw(state):
    """The norm in 64 bits (a long sum), the rest in 32."""
    case, (b1, b2) = state["case"], BETAS
    state["steps"] += 1
    t = state["steps"]
    norm = torch.sqrt(state["grad"].double().square().sum())
    coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
    size, root = LR / (1 - b1 ** t), (1 - b2 ** t) ** 0.5
    first, second = state["first"].split(state["sizes"]), state["second"].split(state["sizes"])
    for i, (p, m, v) in enumerate(zip(state["params"], first, second)):
        g = p.grad.float() * coef
        m.copy_(m * b1 + g * (1 - b1))
        v.copy_(v * b2 + (g * g) * (1 - b2))
        wide = p.detach().float() * (1 - LR * (0.0 if i % 2 else 0.1))
        p.detach().copy_(wide - size * (m / (torch.sqrt(v) / root + EPS)))
        if case["bits"] == 8:
            m.copy_(_held_first(m))
            v.copy_(_held_second(v))
    if case["bits"] == 32:
        return {"params": state["flat"], "first": state["first"], "second": state["second"]}
    # what 8 bits hold has few enough bits for bfloat16 to give back unchanged
    return {"params": state["flat"], "first": [m.bfloat16() for m in first],
            "second": [v.bfloat16() for v in second]}


def _scan(a, b):
    """h_t = a_t h_(t - 1) + b_t along dimension 1 from h = 0, by doubling: after each pass an
    entry stands for twice as many steps."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat((b[:, :step], a[:, step:] * b[:, :-step] + b[:, step:]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def _plain_recurrence(state):
    case = state["case"]
    x, g, h0 = (state[k].detach().float() for k in ("x", "gate", "state"))
    b = x if case["form"] == "add" else (1 - g) * x
    b = torch.cat((b[:, :1] + g[:, :1] * h0[:, None], b[:, 1:]), 1)
    h = _scan(g, b)
    dtype = state["x"].dtype
    out = {"y": h.to(dtype), "last": h[:, -1]}
    if not case["train"]:
        return out
    # dh_t = gy_t + g_(t + 1) dh_(t + 1), the last step also has the last state's gradient
    gy = state["gy"].float()
    gy = torch.cat((gy[:, :-1], gy[:, -1:] + state["gs"][:, None]), 1)
    after = torch.cat((g[:, 1:], torch.zeros_like(g[:, :1])), 1)
    dh = _scan(after.flip(1), gy.flip(1)).flip(1)
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    if case["form"] == "add":
        gx, gg = dh, dh * before
    else:
        gx, gg = dh * (1 - g), dh * (before - x)
    return {**out, "grad_x": gx.to(dtype), "grad_gate": gg.to(dtype), "grad_state": g[:, 0] * dh[:, 0]}


def _plain_verify(state):
    """In 64 bits: sums over the vocabulary, and values next to a border."""
    k = state["case"]["drafts"]
    z, tokens, u = state["logits"].double(), state["tokens"], state["uniforms"].double()
    e = torch.exp(z - z.amax(2, keepdim=True))
    p = e / e.sum(2, keepdim=True)
    e = torch.exp(state["draft"].double() - state["draft"].double().amax(2, keepdim=True))
    q = e / e.sum(2, keepdim=True)
    given = tokens != IGNORE
    at = torch.where(given, tokens, 0)[:, :, None]
    pt, qt = p[:, :k].gather(2, at)[:, :, 0], q.gather(2, at)[:, :, 0]
    good = given & (u[:, :k] * qt < pt)
    accepted = good.long().cumprod(1).sum(1)
    row = torch.arange(len(p), device=p.device)
    # one token more: of what the target has over the draft where a draft was refused, of the
    # target's own probabilities where none was left
    refused = torch.cat((given, torch.zeros_like(given[:, :1])), 1)[row, accepted]
    over = (p[row, accepted] - q[row, accepted.clamp(max=k - 1)]).clamp(min=0)
    weights = torch.where(refused[:, None], over, p[row, accepted])
    sums = weights.cumsum(1)
    last = (sums <= u[:, k:] * sums[:, -1:]).sum(1)
    place = torch.arange(k + 1, device=p.device)
    padded = torch.cat((at[:, :, 0], last[:, None]), 1)
    result = torch.where(place < accepted[:, None], padded, last[:, None])
    lp = torch.log(p.gather(2, result[:, :, None])[:, :, 0])
    behind = place > accepted[:, None]
    return {"tokens": result.masked_fill(behind, IGNORE), "accepted": accepted,
            "log_probs": lp.masked_fill(behind, 0.0).float()}


_PLAIN = {"adamw": _plain_adamw, "recurrence": _plain_recurrence, "verify": _plain_verify}
_OWN = {"adamw": _own_adamw, "recurrence": _own_recurrence, "verify": _own_verify}


# ------------------------------------------------------------------------------------ work

def work(case):
    """Bytes: inputs read once, outputs written once.  Operations per element: adamw 17; the
    recurrence two or four forward and seven or nine more backward; verify a difference, an
    exponential and a sum per logit, and the draw's difference and sum over one row."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "adamw":
        n = sum(_sizes(case))
        moments = 16 if case["bits"] == 32 else 4 + 4  # the latter also given back in bfloat16
        return {"bytes": n * (3 * size + moments), "flops": 17 * n}
    if case["kind"] == "recurrence":
        n = case["batch"] * case["time"] * case["features"]
        states = 4 * case["batch"] * case["features"]
        mix = 2 * (case["form"] == "mix")
        if not case["train"]:
            return {"bytes": 3 * n * size + 2 * states, "flops": (2 + mix) * n}
        return {"bytes": 6 * n * size + 4 * states, "flops": (9 + 2 * mix) * n}
    s, k, v = case["sequences"], case["drafts"], case["vocab"]
    n = s * (2 * k + 1) * v
    return {"bytes": n * size + s * (8 * k + 4 * (k + 1) + 12 * (k + 1) + 8),
            "flops": 3 * n + 4 * s * v}


# ------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return {"adamw": _exact_adamw, "recurrence": _exact_recurrence,
            "verify": _exact_verify}[case["kind"]](state)


def _round_mantissa(x, bits, lowest):
    """x (64 bits) to so many mantissa bits behind the leading one, ties to even; multiples of
    2^(lowest - bits) below 2^lowest."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -1000)))
    e = torch.where(torch.exp2(e) > x.abs(), e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= x.abs(), e + 1, e).clamp(min=lowest)
    unit = torch.exp2(e - bits)
    return torch.round(x / unit) * unit


def _exact_blocks(t, largest_exponent):
    """(rows of a block each, their powers of two, such that the largest lies under
    2^(largest_exponent + 1))."""
    rows = -(-t.numel() // BLOCK)
    b = t.new_zeros(rows * BLOCK)
    b[:t.numel()] = t
    b = b.reshape(rows, BLOCK)
    _, e = torch.frexp(b.abs().max(1, keepdim=True).values)
    return b, torch.exp2((e - 1 - largest_exponent).double())


def _exact_adamw(state):
    case, (b1, b2), t = state["case"], BETAS, STEPS_BEFORE + 1
    norm = torch.linalg.vector_norm(state["grad"].double())
    scale = min(1.0, MAX_NORM / (float(norm) + 1e-6))
    out = {"params": [], "first": [], "second": []}
    parts = [state[k].double().split(state["sizes"]) for k in ("flat", "grad", "first", "second")]
    for i, (p, g, m, v) in enumerate(zip(*parts)):
        g = g * scale
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g.square(), v, b2)
        decay = 0.1 if i % 2 == 0 else 0.0
        p = p - LR * decay * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
        if case["bits"] == 8:
            b, unit = _exact_blocks(m, 7)
            m = (_round_mantissa(b / unit, 3, -6) * unit).reshape(-1)[:m.numel()]
            b, unit = _exact_blocks(v, 0)
            held = _round_mantissa(b / unit, 3, -40)
            held = torch.where(b > 0, held.clamp(min=1.375 * 2.0 ** -31), 0.0)
            v = (held * unit).reshape(-1)[:v.numel()]
        out["params"].append(p)
        out["first"].append(m)
        out["second"].append(v)
    out["params"] = torch.cat(out["params"])
    if case["bits"] == 32:
        out["first"], out["second"] = torch.cat(out["first"]), torch.cat(out["second"])
    return out


def _exact_recurrence(state):
    """Step by step."""
    case = state["case"]
    x, g, h0, gy, gs = (state[k].detach().double() for k in ("x", "gate", "state", "gy", "gs"))
    mix, steps = case["form"] == "mix", case["time"]
    x, g, gy = (t.transpose(0, 1).contiguous() for t in (x, g, gy))
    h = torch.empty_like(x)
    now = h0
    for t in range(steps):
        now = x[t] + g[t] * (now - x[t]) if mix else torch.addcmul(x[t], g[t], now)
        h[t] = now
    out = {"y": h.transpose(0, 1), "last": now}
    if not case["train"]:
        return out
    gx, gg, back = torch.empty_like(x), torch.empty_like(g), gs
    for t in range(steps - 1, -1, -1):
        whole = gy[t] + back
        before = h[t - 1] if t else h0
        gx[t] = whole - g[t] * whole if mix else whole
        gg[t] = (before - x[t]) * whole if mix else before * whole
        back = g[t] * whole
    return {**out, "grad_x": gx.transpose(0, 1), "grad_gate": gg.transpose(0, 1), "grad_state": back}


def _exact_verify(state):
    """Sequence by sequence, drafted token by drafted token."""
    tokens, accepted, log_probs = [], [], []
    k = state["case"]["drafts"]
    drafted, u = state["tokens"].tolist(), state["uniforms"].double().tolist()
    for s, given in enumerate(drafted):
        p = torch.log_softmax(state["logits"][s].double(), 1)
        q = torch.softmax(state["draft"][s].double(), 1)
        result, n = [], 0
        weights = None
        for i, token in enumerate(given):
            if token == IGNORE:
                break
            if not u[s][i] * float(q[i, token]) < float(p[i, token].exp()):
                weights = torch.relu(p[i].exp() - q[i])
                break
            result.append(token)
            n += 1
        if weights is None:
            weights = p[n].exp()
        sums = torch.cumsum(weights, 0)
        result.append(int(torch.searchsorted(sums, u[s][k] * sums[-1], right=True)))
        log_probs.append([float(p[i, t]) for i, t in enumerate(result)] + [0.0] * (k - n))
        tokens.append(result + [IGNORE] * (k - n))
        accepted.append(n)
    return {"tokens": torch.tensor(tokens, device="cuda"), "accepted": torch.tensor(accepted, device="cuda"),
            "log_probs": torch.tensor(log_probs, dtype=torch.float64, device="cuda")}
