"""The operators over class scores and class probabilities: what is measured of them.

A teacher's top logits are selected (`top`), a student is trained on them (`loss`, `grad`), and what
the student drafts is verified against the teacher's probabilities (`verify`). Every case names one
operator, the type of its scores, and its sizes; `layout` says whether a row's classes stand next to
each other ("rows", as a language model's logits do) or a class's rows do ("classes", as a booster's
raw scores do).
"""
import math

import torch

own = False

_TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16,
          "bf16": torch.bfloat16}
_SIZE = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}

# the largest listed gradient moves 2 x 2^28 values of two bytes
_MAX_BYTES = 1 << 29


def _top(name, dtype, layout, rows, classes, k, temperature):
    return {"name": name, "op": "top", "type": dtype, "layout": layout, "rows": rows,
            "classes": classes, "k": k, "temperature": temperature}


def _distill(name, op, dtype, layout, rows, classes, k, temperature, alpha, rest, masked, hessian):
    return {"name": name, "op": op, "type": dtype, "layout": layout, "rows": rows,
            "classes": classes, "k": k, "temperature": temperature, "alpha": alpha,
            "rest": rest, "masked": masked, "hessian": hessian}


def _verify(name, dtype, rows, drafts, classes, with_q, ragged):
    return {"name": name, "op": "verify", "type": dtype, "rows": rows, "drafts": drafts,
            "classes": classes, "with_q": with_q, "ragged": ragged}


def listed():
    return [
        # the answers of one small request are logged with their 20 best classes: latency counts
        _top("top_request", "f32", "rows", 4, 131072, 20, 1.0),
        # a teacher labels a batch of a corpus; an odd number of classes, so rows start at any byte
        _top("top_corpus", "bf16", "rows", 4096, 50021, 64, 2.0),
        # a booster of ten classes labels a million rows of its training data
        _top("top_booster", "f64", "classes", 1000000, 10, 4, 1.0),
        # the evaluation of a student after an epoch, on a held-out batch
        _distill("loss_eval", "loss", "f32", "rows", 2048, 32768, 50, 2.0, 1.0, True, False, False),
        # the same where classes are masked, rows are padding and labels are mixed in
        _distill("loss_masked", "loss", "f16", "rows", 3001, 20011, 17, 1.5, 0.5, True, True, False),
        # a student with a few classes, a small batch: latency counts
        _distill("grad_small", "grad", "f32", "rows", 16, 1000, 8, 1.0, 1.0, False, False, False),
        # one training step of a language model's student
        _distill("grad_tokens", "grad", "bf16", "rows", 8192, 32768, 64, 2.0, 1.0, True, False,
                 False),
        # the same with more classes than a compute unit holds, odd rows and half of the loss on labels
        _distill("grad_wide", "grad", "f32", "rows", 501, 131077, 100, 1.0, 0.5, True, True, False),
        # one boosting iteration: two million rows of seven classes, with hessians
        _distill("grad_booster", "grad", "f64", "classes", 2000000, 7, 3, 2.0, 0.7, True, True,
                 True),
        # one sequence of four drafts is verified: latency counts
        _verify("verify_one", "f32", 1, 4, 131072, True, False),
        # a serving batch, sequences with fewer drafts among them
        _verify("verify_batch", "bf16", 256, 7, 50021, True, True),
        # answers drafted by a student of ten classes without probabilities (its best class)
        _verify("verify_booster", "f64", 100000, 3, 10, False, True),
    ]


def _spread(rng, lo, hi):
    """A whole number, spread over the logarithm of lo..hi; every other one made odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v |= 1
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["top", "loss", "grad", "verify"])
    if op == "verify":
        dtype = rng.choice(["f64", "f32", "f16", "bf16"])
        drafts = rng.randint(1, 8)
        classes = _spread(rng, 2, 200000)
        # the target's and the draft's probabilities together
        most = _MAX_BYTES // (_SIZE[dtype] * classes * (2 * drafts + 1))
        rows = _spread(rng, 1, max(1, min(most, 200000)))
        return {"op": op, "type": dtype, "rows": rows, "drafts": drafts, "classes": classes,
                "with_q": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    booster = rng.random() < 0.35
    if booster:
        dtype = rng.choice(["f64", "f64", "f32"])
        layout = "classes"
        classes = _spread(rng, 3, 300)
    else:
        dtype = rng.choice(["f32", "f16", "bf16"])
        layout = "rows"
        classes = _spread(rng, 3, 200000)
    most = _MAX_BYTES // (2 * _SIZE[dtype] * classes)
    rows = _spread(rng, 1, max(1, min(most, 2000000)))
    k = min(_spread(rng, 1, 200), max(1, classes // 2))
    case = {"op": op, "type": dtype, "layout": layout, "rows": rows, "classes": classes, "k": k,
            "temperature": rng.choice([1.0, 1.0, 1.5, 2.0, 4.0])}
    if op != "top":
        case["alpha"] = rng.choice([1.0, 1.0, 0.5, 0.9])
        case["rest"] = rng.random() < 0.6
        case["masked"] = rng.random() < 0.5
        case["hessian"] = op == "grad" and booster
    return case


# ------------------------------------------------------------------ inputs
def _scores(case, g, dtype):
    """Class scores [rows, classes] in the case's layout: a broad bulk, and in every row a few
    classes that stand out."""
    n, c = case["rows"], case["classes"]
    shape = (c, n) if case["layout"] == "classes" else (n, c)
    x = torch.randn(shape, generator=g, device="cuda")
    x = x.t() if case["layout"] == "classes" else x
    top = min(8, c)
    step = c // top
    best = torch.randint(0, c, (n, 1), generator=g, device="cuda")
    best = (best + step * torch.arange(top, device="cuda")
            + torch.randint(0, step, (n, top), generator=g, device="cuda")) % c
    lift = 6.0 * torch.rand((n, top), generator=g, device="cuda")
    x.scatter_add_(1, best, lift)
    return x.to(dtype)


def _teacher(case, g):
    """Top classes without repeats, descending logits, and the logarithm of what is left."""
    n, c, k = case["rows"], case["classes"], case["k"]
    step = c // k
    at = torch.arange(k, device="cuda") * step
    jitter = torch.randint(0, step, (n, k), generator=g, device="cuda")
    start = torch.randint(0, c, (n, 1), generator=g, device="cuda")
    classes = (start + at + jitter) % c
    logits = (8.0 * torch.rand((n, k), generator=g, device="cuda")).sort(1, descending=True)[0]
    rest = 1.0 + 4.0 * torch.rand(n, generator=g, device="cuda") if case["rest"] else None
    if case["masked"]:
        # every 16th row has a shorter list, every 64th none at all
        row = torch.arange(n, device="cuda")[:, None]
        slot = torch.arange(k, device="cuda")[None, :]
        gone = ((row % 16 == 3) & (slot >= (k + 1) // 2)) | (row % 64 == 7)
        classes = classes.masked_fill(gone, -1)
        logits = logits.masked_fill(gone, -math.inf)
        if rest is not None:
            rest = rest.masked_fill((row % 64 == 7)[:, 0], -math.inf)
    return classes.int(), logits, rest


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "top":
        state["scores"] = _scores(case, g, dtype)
        return state
    if case["op"] == "verify":
        b, t, c = case["rows"], case["drafts"], case["classes"]
        x = 2.0 * torch.randn((b, t + 1, c), generator=g, device="cuda")
        # the draft's scores are the target's with noise, so that most drafts are accepted
        y = x[:, :t] + 0.5 * torch.randn((b, t, c), generator=g, device="cuda")
        state["target"] = torch.softmax(x, 2).to(dtype)
        q = torch.softmax(y, 2).to(dtype)
        # classes drawn from q: the smallest of c exponential clocks with rates q
        clock = torch.empty_like(y).exponential_(generator=g)
        pick = (q.float() / clock).argmax(2) if case["with_q"] else q.float().argmax(2)
        state["drafts"] = pick.int()
        state["draft"] = q if case["with_q"] else None
        state["accept"] = torch.rand((b, t), generator=g, device="cuda")
        state["sample"] = torch.rand((b,), generator=g, device="cuda")
        state["lengths"] = (torch.randint(0, t + 1, (b,), generator=g, device="cuda").int()
                            if case["ragged"] else None)
        return state
    scores = _scores(case, g, dtype)
    n, c = case["rows"], case["classes"]
    classes, logits, rest = _teacher(case, g)
    state["labels"] = None
    state["weight"] = None
    if case["alpha"] != 1.0:
        state["labels"] = torch.randint(0, c, (n,), generator=g, device="cuda").int()
    if case["masked"]:
        # one class in 32 is not allowed where there are many, unless the teacher or the label
        # names it
        bar = torch.rand((n, c), generator=g, device="cuda") < (1 / 32 if c >= 64 else 0)
        at = classes.long().clamp(0)
        bar.scatter_(1, at, False)
        if state["labels"] is not None:
            bar.scatter_(1, state["labels"].long()[:, None], False)
        scores.masked_fill_(bar, -math.inf)
        # padding rows have no weight
        weight = 0.5 + torch.rand((n,), generator=g, device="cuda")
        weight[torch.arange(n, device="cuda") % 8 == 5] = 0.0
        state["weight"] = weight
    state["scores"] = scores
    state["classes"], state["logits"], state["rest"] = classes, logits, rest
    return state


# ------------------------------------------------------------------ plain forms
def _plain_top(state):
    case = state["case"]
    x = state["scores"]
    # raw scores of a booster are 64 bits: 32 would make ties of neighbours
    wide = x if x.dtype == torch.float64 else x.float()
    values, order = torch.sort(wide, dim=1, descending=True, stable=True)
    k = case["k"]
    left = values[:, k:] / case["temperature"]
    high = left[:, :1]
    rest = torch.log(torch.exp(left - high).sum(1)) + high[:, 0]
    return order[:, :k].int(), values[:, :k].to(x.dtype), rest


def _plain_distill(state):
    case = state["case"]
    z = state["scores"]
    wide = torch.float64 if z.dtype == torch.float64 else torch.float32
    x = z.to(wide)
    n, c = z.shape
    t, alpha = case["temperature"], case["alpha"]
    valid = state["classes"] >= 0
    at = state["classes"].long().clamp(0)
    slot = torch.where(valid, state["logits"].to(wide) / t, -math.inf)
    if state["rest"] is not None:
        slot = torch.cat([slot, (state["rest"].to(wide))[:, None]], 1)
    high = slot.amax(1, keepdim=True)
    there = (high > -math.inf)
    soft = torch.exp(slot - torch.where(there, high, 0.0))
    soft = soft / soft.sum(1, keepdim=True).clamp_min(1e-30)
    p, r = soft[:, :case["k"]], soft[:, case["k"]:]

    s = x / t
    top = s.amax(1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(1, keepdim=True)
    log_q = torch.gather(s, 1, at) - top - torch.log(total)
    # what the student gives to the classes that the teacher does not name
    named = torch.zeros((n, c + 1), dtype=torch.bool, device=z.device)
    named.scatter_(1, torch.where(valid, at, c), True)
    named = named[:, :c]
    left = torch.where(named, 0.0, e).sum(1, keepdim=True)
    weight = 1.0 if state["weight"] is None else state["weight"].to(wide)[:, None]
    labels = state["labels"]
    if labels is not None:
        y = labels.long()[:, None]
        high1 = x.amax(1, keepdim=True)
        e1 = torch.exp(x - high1)
        total1 = e1.sum(1, keepdim=True)
    if case["op"] == "loss" or not case["hessian"]:
        kl = torch.where(p > 0, p * (torch.log(p.clamp_min(1e-38)) - log_q), 0.0).sum(1, True)
        if state["rest"] is not None:
            log_rho = torch.log(left) - torch.log(total)
            kl = kl + torch.where(r > 0, r * (torch.log(r.clamp_min(1e-38)) - log_rho), 0.0)
        loss = alpha * t * t * torch.where(there, kl, 0.0)
        if labels is not None:
            hard = torch.log(total1) + high1 - torch.gather(x, 1, y)
            loss = loss + (1 - alpha) * hard
        loss = (loss * weight)[:, 0]
        if case["op"] == "loss":
            return loss
    q = e / total
    want = torch.zeros((n, c + 1), dtype=wide, device=z.device)
    if state["rest"] is not None:
        want[:, :c] = torch.where(named, 0.0, e) * (r / left)
    want.scatter_(1, torch.where(valid, at, c), p)
    grad = torch.where(there, alpha * t * (q - want[:, :c]), 0.0)
    if labels is not None:
        p1 = e1 / total1
        one = torch.arange(c, device=z.device)[None, :] == y
        grad = grad + (1 - alpha) * (p1 - one.to(wide))
    out = torch.float32 if z.dtype == torch.float64 else z.dtype
    grad = (grad * weight).to(out)
    if not case["hessian"]:
        return grad, loss
    hess = torch.where(there, alpha * q * (1 - q), 0.0)
    if labels is not None:
        hess = hess + (1 - alpha) * p1 * (1 - p1)
    return grad, (hess * weight * (c / (c - 1))).to(out)


def _plain_verify(state):
    p = state["target"]
    b, t1, c = p.shape
    t = t1 - 1
    x = state["drafts"].long()
    step = torch.arange(t, device=p.device)[None, :]
    lengths = (state["lengths"].long()[:, None] if state["lengths"] is not None
               else torch.full((b, 1), t, device=p.device))
    # 64 bits: a draft or a draw may stand next to a border
    p_x = torch.gather(p[:, :t], 2, x[:, :, None])[:, :, 0].double()
    if state["draft"] is not None:
        q_x = torch.gather(state["draft"], 2, x[:, :, None])[:, :, 0].double()
    else:
        q_x = torch.ones_like(p_x)
    good = (state["accept"].double() * q_x < p_x) & (step < lengths)
    accepted = torch.cumprod(good.long(), 1).sum(1)
    row = torch.arange(b, device=p.device)
    left = p[row, accepted].double()
    refused = accepted < lengths[:, 0]
    last = accepted.clamp_max(t - 1)
    if state["draft"] is not None:
        less = state["draft"][row, last].double()
    else:
        less = torch.zeros_like(left).scatter_(1, x[row, last][:, None], 1.0)
    left = torch.where(refused[:, None], (left - less).clamp_min(0), left)
    total = torch.cumsum(left, 1)
    drawn = (total > state["sample"].double()[:, None] * total[:, -1:]).long().argmax(1)
    at = torch.arange(t1, device=p.device)[None, :]
    tokens = torch.cat([x, torch.full((b, 1), -1, device=p.device)], 1)
    tokens = torch.where(at < accepted[:, None], tokens, -1)
    tokens = torch.where(at == accepted[:, None], drawn[:, None], tokens)
    return tokens.int(), accepted.int()


def run(state):
    case = state["case"]
    if own:
        from lightgbm_amd import ops
        if case["op"] == "top":
            got = ops.top_logits(state["scores"], case["k"], temperature=case["temperature"])
            return got.classes, got.logits, got.log_rest
        if case["op"] == "verify":
            got = ops.verify_drafts(state["target"], state["drafts"], state["draft"],
                                    state["accept"], state["sample"], lengths=state["lengths"])
            return got.classes, got.accepted
        teacher = ops.TopLogits(state["classes"], state["logits"], state["rest"])
        mix = {"labels": state["labels"], "weight": state["weight"],
               "temperature": case["temperature"], "alpha": case["alpha"]}
        if case["op"] == "loss":
            return ops.distill_loss(state["scores"], teacher, **mix)
        if case["hessian"]:
            got = ops.distill_gradients(state["scores"], teacher, hessian=True, **mix)
            return got.gradient, got.hessian
        got = ops.distill_gradients(state["scores"], teacher, loss=True, **mix)
        return got.gradient, got.loss
    if case["op"] == "top":
        return _plain_top(state)
    if case["op"] == "verify":
        return _plain_verify(state)
    return _plain_distill(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n, c, size = case["rows"], case["classes"], _SIZE[case["type"]]
    if case["op"] == "top":
        # one comparison, one scaling, one exponential and one sum for each score
        return {"bytes": n * c * size + n * case["k"] * (size + 4) + n * max(4, size // 2),
                "flops": 4 * n * c}
    if case["op"] == "verify":
        t = case["drafts"]
        # the drafted classes' probabilities, and the one row of each side that the last class is
        # drawn from; one difference and one sum for each of its classes
        sides = 2 if case["with_q"] else 1
        return {"bytes": n * (t * (8 + sides * size) + sides * c * size + 4 * (t + 3)),
                "flops": n * c * (sides + 1)}
    out = 4 if case["type"] == "f64" else size
    moved = n * c * size + n * case["k"] * 8 + n * 16
    # softmax at the temperature, and a second one for the labels
    flops = (4 if case["alpha"] == 1.0 or case["temperature"] == 1.0 else 8) * n * c
    if case["op"] == "grad":
        moved += n * c * out * (2 if case["hessian"] else 1)
        flops += (7 if case["hessian"] else 3) * n * c
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ from the definitions, 64 bits
def _exact_top(state):
    case = state["case"]
    classes, logits, rest = [], [], []
    k, t = case["k"], case["temperature"]
    c = case["classes"]
    for x in torch.split(state["scores"], max(1, (1 << 25) // c)):
        x = x.contiguous().double()
        # the k-th largest value: all above it are chosen, and of its equals the lowest classes
        edge = x.topk(k, 1)[0][:, -1:]
        above = x > edge
        equal = x == edge
        chosen = above | (equal & (equal.int().cumsum(1) <= k - above.sum(1, True)))
        at = chosen.nonzero()[:, 1].view(-1, k)
        value = x.gather(1, at)
        order = torch.argsort(value, dim=1, descending=True, stable=True)
        classes.append(at.gather(1, order).int())
        logits.append(value.gather(1, order))
        rest.append(torch.logsumexp((x / t).masked_fill(chosen, -math.inf), 1))
    return torch.cat(classes), torch.cat(logits), torch.cat(rest)


def _exact_distill(state):
    case = state["case"]
    t, alpha, c, k = case["temperature"], case["alpha"], case["classes"], case["k"]
    inf = math.inf
    found = []
    step = max(1, (1 << 25) // c)
    for i in range(0, case["rows"], step):
        part = slice(i, i + step)
        x = state["scores"][part].contiguous().double()
        n = x.shape[0]
        log_q = torch.log_softmax(x / t, 1)
        at = state["classes"][part].long()
        logit = torch.where(at >= 0, state["logits"][part].double() / t, -inf)
        rest = (state["rest"][part].double() if state["rest"] is not None
                else torch.full((n,), -inf, dtype=torch.float64, device=x.device))
        norm = torch.logaddexp(torch.logsumexp(logit, 1), rest)
        some = norm > -inf
        norm = torch.where(some, norm, 0.0)
        # the target's logarithm over all classes: the slots, and the rest shared out as the student has it
        other = log_q.clone()
        rows, slots = (at >= 0).nonzero(as_tuple=True)
        other[rows, at[rows, slots]] = -inf
        log_rho = torch.logsumexp(other, 1)
        target = torch.exp(other + (rest - norm - log_rho)[:, None])
        target[rows, at[rows, slots]] = torch.exp(logit[rows, slots] - norm[rows])
        w = (state["weight"][part].double() if state["weight"] is not None
             else torch.ones(n, dtype=torch.float64, device=x.device))
        soft = some.double() * alpha
        hard = 1 - alpha
        loss = torch.zeros(n, dtype=torch.float64, device=x.device)
        log_p = logit[rows, slots] - norm[rows]
        term = torch.exp(log_p) * (log_p - log_q[rows, at[rows, slots]])
        loss.index_add_(0, rows, torch.where(log_p > -inf, term, 0.0))
        share = torch.exp(rest - norm)
        loss += torch.where(rest > -inf, share * (rest - norm - log_rho), 0.0)
        loss = loss * soft * t * t
        gradient = (soft * t)[:, None] * (torch.exp(log_q) - target)
        q = torch.exp(log_q)
        curve = soft[:, None] * (q - q * q)
        if state["labels"] is not None:
            y = state["labels"][part].long()
            log_1 = torch.log_softmax(x, 1)
            here = torch.arange(n, device=x.device)
            loss += hard * -log_1[here, y]
            p1 = torch.exp(log_1)
            curve += hard * (p1 - p1 * p1)
            p1[here, y] -= 1.0
            gradient += hard * p1
        if case["op"] == "loss":
            found.append((loss * w,))
        elif case["hessian"]:
            found.append((gradient * w[:, None], curve * w[:, None] * c / (c - 1)))
        else:
            found.append((gradient * w[:, None], loss * w))
    return tuple(torch.cat(parts) for parts in zip(*found))


def _exact_verify(state):
    p = state["target"]
    b, t1, c = p.shape
    t = t1 - 1
    x = state["drafts"].long().cpu()
    lengths = state["lengths"].cpu() if state["lengths"] is not None else torch.full((b,), t)
    u = state["accept"].double().cpu()
    at = state["drafts"].long()[:, :, None]
    p_x = p[:, :t].gather(2, at)[:, :, 0].double().cpu()
    q_x = (state["draft"].gather(2, at)[:, :, 0].double().cpu() if state["draft"] is not None
           else torch.ones_like(p_x))
    accepted = torch.zeros(b, dtype=torch.long)
    going = torch.ones(b, dtype=torch.bool)
    for i in range(t):
        going &= (i < lengths) & (u[:, i] * q_x[:, i] < p_x[:, i])
        accepted += going
    tokens = torch.full((b, t1), -1, dtype=torch.long)
    for i in range(t):
        tokens[:, i] = torch.where(accepted > i, x[:, i], tokens[:, i])
    v = state["sample"].double()
    drawn = []
    for i in range(0, b, 8192):
        rows = torch.arange(i, min(i + 8192, b))
        a = accepted[rows]
        mass = p[rows.to(p.device), a.to(p.device)].double()
        full = (a < lengths[rows]).to(p.device)
        j = a.clamp_max(t - 1).to(p.device)
        if state["draft"] is not None:
            mass -= torch.where(full[:, None], state["draft"][rows.to(p.device), j].double(), 0.0)
        else:
            refused = state["drafts"].long()[rows.to(p.device), j]
            here = torch.arange(len(rows), device=p.device)
            mass[here, refused] -= full.double()
        mass = mass.clamp(min=0.0)
        reach = mass.cumsum(1)
        goal = v[rows.to(p.device)] * reach[:, -1]
        drawn.append(torch.searchsorted(reach, goal[:, None], right=True)[:, 0])
    tokens[torch.arange(b), accepted] = torch.cat(drawn).cpu()
    return tokens.int().to(p.device), accepted.int().to(p.device)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "top":
        return _exact_top(state)
    if case["op"] == "verify":
        return _exact_verify(state)
    found = _exact_distill(state)
    return found[0] if case["op"] == "loss" else found
