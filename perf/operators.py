"""What the operators on two models' class distributions are measured on: the k largest logits of every row
(``ops.top_logits``), distillation from them (``criterions.distill_top_loss``) and the verification of drafted
classes (``ops.verify_drafts``), each with a plain form in elementary torch operations.

A row is one token's logits over a vocabulary, or one voxel's over a segmentation model's classes.
``own = False`` runs the plain forms, ``own = True`` the framework's kernels.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "bf16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a served teacher: a single row, latency
        dict(name="top_one_row", op="top", rows=1, classes=32768, k=8, type="bf16", layout="last", space="",
             rest=True, temperature=1.0),
        # a teacher's pass over a batch of long sequences, kept as its 64 largest logits a token
        dict(name="top_vocabulary", op="top", rows=2048, classes=131072, k=64, type="bf16", layout="last", space="",
             rest=True, temperature=2.0),
        # a segmentation teacher's two largest class logits of every voxel of a training batch
        dict(name="top_volume", op="top", rows=2, classes=4, k=2, type="fp32", layout="last", space="128x128x128",
             rest=True, temperature=2.0),
        # a training step on a handful of tokens (the last, short micro-batch): latency of loss and gradient
        dict(name="distill_few_rows", op="distill", rows=16, classes=32768, k=16, type="fp32", layout="last", space="",
             rest=True, mask=False, temperature=2.0, gradient=True),
        # the ordinary large step: 4096 tokens against a large vocabulary, with the mass outside the top as one class
        dict(name="distill_vocabulary", op="distill", rows=4096, classes=131072, k=64, type="bf16", layout="last",
             space="", rest=True, mask=False, temperature=2.0, gradient=True),
        # an odd vocabulary (rows start at any alignment), padded tokens masked, the top renormalised
        dict(name="distill_odd_masked", op="distill", rows=1021, classes=50001, k=20, type="bf16", layout="last",
             space="", rest=False, mask=True, temperature=1.0, gradient=True),
        # the loss of every token alone, as an evaluation pass computes it
        dict(name="distill_loss_only", op="distill", rows=1500, classes=32001, k=32, type="fp32", layout="last",
             space="", rest=True, mask=False, temperature=1.0, gradient=False),
        # the U-Net's training batch: channels-last voxels, two of four classes kept
        dict(name="distill_volume", op="distill", rows=2, classes=4, k=2, type="bf16", layout="last",
             space="128x128x128", rest=True, mask=False, temperature=2.0, gradient=True),
        # a 2-D batch of seven classes, channels first
        dict(name="distill_images_first", op="distill", rows=8, classes=7, k=3, type="fp32", layout="first",
             space="512x512", rest=True, mask=True, temperature=2.0, gradient=True),
        # one served sequence with four drafted tokens: latency
        dict(name="verify_one_sequence", op="verify", rows=1, drafts=4, classes=32768, type="fp32", drafter=True,
             bonus=True, ragged=False),
        # a serving batch: ragged draft lengths, a large vocabulary
        dict(name="verify_batch", op="verify", rows=200, drafts=7, classes=131072, type="bf16", drafter=True,
             bonus=True, ragged=True),
        # label maps: every voxel's drafted class against the target's four probabilities
        dict(name="verify_volume", op="verify", rows=128 ** 3, drafts=1, classes=4, type="fp32", drafter=True,
             bonus=False, ragged=False),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["top", "distill", "distill", "verify"])
    kind = rng.choice(["vocabulary", "vocabulary", "voxels"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "verify":
        if kind == "voxels":
            return dict(op=op, rows=_log(rng, 1000, 128 ** 3), drafts=1, classes=rng.randint(2, 10), type=dtype,
                        drafter=rng.random() < 0.7, bonus=False, ragged=False)
        classes = _log(rng, 1000, 131072)
        drafts = rng.randint(1, 8)
        most = max(1, min(256, 120_000_000 // (classes * drafts)))
        return dict(op=op, rows=_log(rng, 1, most), drafts=drafts, classes=classes, type=dtype,
                    drafter=rng.random() < 0.7, bonus=rng.random() < 0.7, ragged=rng.random() < 0.5)
    case = dict(op=op, type=dtype, rest=rng.random() < 0.7, temperature=rng.choice([1.0, 1.5, 2.0, 4.0]))
    if kind == "voxels":
        classes = rng.randint(2, 10)
        case.update(rows=rng.randint(1, 4), classes=classes, k=rng.randint(1, classes),
                    layout=rng.choice(["first", "last"]),
                    space="x".join(str(_log(rng, 8, 96)) for _ in range(3)))
    else:
        classes = _log(rng, 1000, 131072)
        most = max(1, min(4096, 200_000_000 // classes))
        case.update(rows=_log(rng, 1, most), classes=classes, k=_log(rng, 1, 100), layout="last", space="")
    if op == "distill":
        case.update(mask=rng.random() < 0.5, gradient=rng.random() < 0.75)
    return case


def _space(case):
    return [int(s) for s in case["space"].split("x") if s]


def _voxels(case):
    return case["rows"] * math.prod(_space(case))


def work(case):
    e, classes = _SIZE[case["type"]], case["classes"]
    if case["op"] == "verify":
        rows, drafts = case["rows"], case["drafts"]
        models = 2 if case["drafter"] else 1
        # one row of each model's probabilities a sequence; drafted tokens, their probabilities and random numbers
        read = rows * (models * classes * e + drafts * (8 + 4 + models * e) + 4)
        return {"bytes": read + rows * (drafts + int(case["bonus"]) + 1) * 8, "flops": 3 * rows * classes}
    n, k = _voxels(case), case["k"]
    top = n * (k * (e + (1 if classes <= 256 else 4)) + (4 if case["rest"] else 0))
    if case["op"] == "top":
        return {"bytes": n * classes * e + top, "flops": 4 * n * classes}
    mask = n if case["mask"] else 0
    if case["gradient"]:
        return {"bytes": 2 * n * classes * e + top + mask + 4, "flops": 8 * n * classes}
    return {"bytes": n * classes * e + top + mask + 4 * n, "flops": 4 * n * classes}


# ------------------------------------------------------------------ inputs
def _first(x, case):
    """(rows, *space, c) as the case lays it out."""
    return x.movedim(-1, 1).contiguous() if case["layout"] == "first" else x


def _last(x, case):
    return x.movedim(1, -1) if case["layout"] == "first" else x


def _normal(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]
    if case["op"] == "verify":
        return _prepare_verify(case, g, kind)
    shape = (case["rows"], *_space(case), case["classes"])
    # a trained model's logits: a wide bell and a few classes that stand out, which together hold most of the mass
    logits = _normal(shape, g).mul_(2.0)
    some = max(1, min(16, case["classes"] // 8))
    peak = torch.randint(0, case["classes"], shape[:-1] + (some,), generator=g, device="cuda")
    high = math.log(case["classes"]) * (0.5 + torch.rand(peak.shape, generator=g, device="cuda"))
    logits.scatter_add_(-1, peak, high.add_(torch.rand(peak.shape, generator=g, device="cuda"), alpha=4.0))
    del peak, high
    state = {"case": case}
    if case["op"] == "top":
        state["logits"] = _first(logits, case).to(kind)
        return state
    # the student is the teacher, some way off
    student = _first(logits + _normal(shape, g), case).to(kind)
    teacher = logits.to(kind)
    values, order = torch.topk(teacher, case["k"], dim=-1)
    state["values"] = _first(values, case)
    state["indices"] = _first(order, case).to(torch.uint8 if case["classes"] <= 256 else torch.int32)
    state["rest"] = None
    if case["rest"]:
        scaled = teacher.float().div_(case["temperature"]).scatter_(-1, order, -math.inf)
        state["rest"] = torch.logsumexp(scaled, -1)
    # padded tokens, or voxels outside the scanned body
    state["mask"] = torch.rand(shape[:-1], generator=g, device="cuda") < 0.8 if case["mask"] else None
    state["logits"] = student.requires_grad_(case["gradient"])
    return state


def _prepare_verify(case, g, kind):
    rows, drafts, classes = case["rows"], case["drafts"], case["classes"]
    steps = drafts + int(case["bonus"])
    logits = _normal((rows, steps, classes), g).mul_(3.0)
    target = torch.softmax(logits, -1).to(kind)
    draft = torch.softmax(logits[:, :drafts] + 0.7 * _normal((rows, drafts, classes), g), -1).to(kind)
    del logits
    # the drafter's own draws
    place = torch.rand((rows, drafts, 1), generator=g, device="cuda", dtype=torch.float64)
    reach = draft.double().cumsum(-1)
    tokens = torch.searchsorted(reach, place * reach[..., -1:], right=True).squeeze(-1).clamp_(max=classes - 1)
    del reach
    return {"case": case, "tokens": tokens, "target": target, "draft": draft if case["drafter"] else None,
            "accept": torch.rand((rows, drafts), generator=g, device="cuda"),
            "sample": torch.rand((rows,), generator=g, device="cuda"),
            "lengths": torch.randint(0, drafts + 1, (rows,), generator=g, device="cuda") if case["ragged"] else None}


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"top": _own_top, "distill": _own_distill, "verify": _own_verify}[op](state)
    with torch.no_grad():
        return {"top": _plain_top, "distill": _plain_distill, "verify": _plain_verify}[op](state)


def _own_top(state):
    from devis_amd import ops
    case = state["case"]
    out = ops.top_logits(state["logits"], case["k"], channels_last=case["layout"] == "last",
                         temperature=case["temperature"], want_rest=case["rest"])
    return [out["values"], out["indices"], out["rest"]] if case["rest"] else [out["values"], out["indices"]]


def _own_distill(state):
    from devis_amd import criterions
    case = state["case"]
    args = (state["logits"], state["values"], state["indices"])
    kw = dict(rest=state["rest"], channels_last=case["layout"] == "last", temperature=case["temperature"],
              row_mask=state["mask"])
    if not case["gradient"]:
        with torch.no_grad():
            return [criterions.distill_top_loss(*args, reduction="none", **kw)]
    loss = criterions.distill_top_loss(*args, **kw)
    return [loss.detach(), torch.autograd.grad(loss, state["logits"])[0]]


def _own_verify(state):
    from devis_amd import ops
    out = ops.verify_drafts(state["tokens"], state["target"], state["draft"], state["accept"], state["sample"],
                            lengths=state["lengths"])
    return [out["tokens"], out["accepted"]]


# ------------------------------------------------------------------ plain forms
def _plain_top(state):
    case = state["case"]
    logits = _last(state["logits"], case)
    x = logits.float()
    # order by value, then by lowest index: the value's bits as an ordered integer above the index counted downwards
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    code = bits * 2 ** 32 + (case["classes"] - 1 - torch.arange(case["classes"], device=x.device))
    order = torch.topk(code, case["k"], dim=-1)[1]
    del bits, code
    out = [_first(torch.gather(logits, -1, order), case),
           _first(order, case).to(torch.uint8 if case["classes"] <= 256 else torch.int32)]
    if case["rest"]:
        x = (x / case["temperature"]).scatter_(-1, order, -math.inf)
        high = x.max(-1, keepdim=True)[0]
        high = torch.where(high == -math.inf, torch.zeros_like(high), high)
        out.append((torch.exp(x - high).sum(-1, keepdim=True, dtype=torch.float64).log() + high).squeeze(-1).float())
    return out


def _plain_teacher(values, rest, temperature):
    """Shares of the teacher's slots and of the rest, and their logarithms, in 64 bits."""
    t = values.double() / temperature
    if rest is not None:
        t = torch.cat([t, rest.unsqueeze(-1).double()], -1)
    high = t.max(-1, keepdim=True)[0]
    log_p = t - high
    log_p = log_p - torch.exp(log_p).sum(-1, keepdim=True).log()
    return torch.exp(log_p), log_p


def _plain_distill(state):
    case = state["case"]
    temperature, k = case["temperature"], case["k"]
    x = _last(state["logits"], case).float() / temperature
    values, index = _last(state["values"], case), _last(state["indices"], case).long()
    p, log_p = _plain_teacher(values, state["rest"], temperature)
    high = x.max(-1, keepdim=True)[0]
    # the logarithms are near one another where the student is near the teacher: their difference in 64 bits
    lse = torch.exp(x - high).sum(-1, keepdim=True, dtype=torch.float64).log() + high
    log_q = torch.gather(x, -1, index) - lse
    if state["rest"] is not None:
        left = x.scatter(-1, index, -math.inf)
        top = left.max(-1, keepdim=True)[0]
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        lse_left = torch.exp(left - top).sum(-1, keepdim=True, dtype=torch.float64).log() + top
        log_q = torch.cat([log_q, lse_left - lse], -1)
    loss = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(-1) * temperature ** 2
    if state["mask"] is not None:
        loss = torch.where(state["mask"], loss, torch.zeros_like(loss))
    if not case["gradient"]:
        return [loss.float()]
    count = loss.numel() if state["mask"] is None else state["mask"].sum()
    total = (loss.sum() / count).float()
    grad = torch.exp(x - lse.float())
    if state["rest"] is not None:
        left.sub_(lse_left.float()).exp_()
        # no class is left: nothing to share out
        left = torch.where(lse_left == -math.inf, torch.zeros_like(left), left)
        grad.sub_(left.mul_(p[..., k:].float()))
    grad.scatter_add_(-1, index, -p[..., :k].float()).mul_(temperature / count)
    if state["mask"] is not None:
        grad.mul_(state["mask"].unsqueeze(-1))
    return [total, _first(grad, case).to(state["logits"].dtype)]


def _plain_verify(state):
    case, tokens = state["case"], state["tokens"]
    target, draft = state["target"], state["draft"]
    rows, drafts = tokens.shape
    steps = target.shape[1]
    each = torch.arange(rows, device=tokens.device)
    # in 64 bits: products and sums next to a border decide
    p = torch.gather(target[:, :drafts], -1, tokens.unsqueeze(-1)).squeeze(-1).double()
    u = state["accept"].double()
    if draft is not None:
        u = u * torch.gather(draft, -1, tokens.unsqueeze(-1)).squeeze(-1).double()
    place = torch.arange(drafts, device=tokens.device)
    length = torch.full_like(each, drafts) if state["lengths"] is None else state["lengths"]
    good = (u < p) & (place < length[:, None])
    accepted = good.long().cumprod(-1).sum(-1)
    stopped = accepted < length
    at = accepted.clamp(max=steps - 1)
    weight = target[each, at].double()
    whole = weight
    back = accepted.clamp(max=drafts - 1)
    if draft is not None:
        weight = torch.where(stopped[:, None], (weight - draft[each, back].double()).clamp_min(0), weight)
    else:
        weight = torch.where(stopped[:, None] & (torch.arange(case["classes"], device=tokens.device) == tokens[each, back][:, None]),
                             torch.zeros_like(weight), weight)
    weight = torch.where(weight.sum(-1, keepdim=True) > 0, weight, whole)
    reach = weight.cumsum(-1)
    goal = state["sample"].double() * reach[:, -1]
    drawn = (reach <= goal[:, None]).sum(-1)
    last = case["classes"] - 1 - (weight.flip(-1) > 0).to(torch.uint8).argmax(-1)
    drawn = torch.minimum(drawn, last)
    answer = torch.full((rows, steps), -1, dtype=tokens.dtype, device=tokens.device)
    answer[:, :drafts] = torch.where(place < accepted[:, None], tokens, answer[:, :drafts])
    draws = stopped | (accepted < steps)
    answer[each[draws], accepted[draws]] = drawn[draws]
    return [answer, accepted]


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"top": _exact_top, "distill": _exact_distill, "verify": _exact_verify}[case["op"]](case, state)


def _pieces(rows, classes):
    """Ranges of rows of at most 2^26 numbers."""
    step = max(1, 2 ** 26 // classes)
    return [slice(a, min(rows, a + step)) for a in range(0, rows, step)]


def _flat(x, case):
    x = _last(x, case)
    return x.reshape(-1, x.shape[-1])


def _shaped(x, case):
    """(all rows, c) back to the case's layout."""
    return _first(x.reshape(case["rows"], *_space(case), x.shape[-1]), case)


def _exact_top(case, state):
    z = _flat(state["logits"], case)
    values, indices, rest = [], [], []
    for part in _pieces(*z.shape):
        y, order = torch.sort(z[part].double(), dim=-1, descending=True, stable=True)
        values.append(y[:, :case["k"]])
        indices.append(order[:, :case["k"]])
        rest.append(torch.logsumexp(y[:, case["k"]:] / case["temperature"], -1) if case["k"] < case["classes"]
                    else torch.full_like(y[:, 0], -math.inf))
    out = [_shaped(torch.cat(values), case),
           _shaped(torch.cat(indices), case).to(torch.uint8 if case["classes"] <= 256 else torch.int32)]
    if case["rest"]:
        out.append(torch.cat(rest).reshape(case["rows"], *_space(case)))
    return out


def _exact_distill(case, state):
    z, values, indices = (_flat(state[name], case) for name in ("logits", "values", "indices"))
    n, classes = z.shape
    mask = torch.ones(n, dtype=torch.bool, device=z.device) if state["mask"] is None else state["mask"].reshape(-1)
    temperature = case["temperature"]
    losses, grads = [], []
    for part in _pieces(n, classes):
        rows = torch.arange(part.stop - part.start, device=z.device)[:, None]
        index = indices[part].long()
        t = values[part].double() / temperature
        log_q = torch.log_softmax(z[part].double() / temperature, -1)
        listed_too = torch.zeros_like(log_q, dtype=torch.bool)
        listed_too[rows, index] = True
        if state["rest"] is None:
            log_p = torch.log_softmax(t, -1)
            loss = (log_p.exp() * (log_p - log_q[rows, index])).sum(-1)
            wanted = torch.zeros_like(log_q)
        else:
            log_p = torch.log_softmax(torch.cat([t, state["rest"].reshape(-1)[part, None].double()], -1), -1)
            outside = log_q.masked_fill(listed_too, -math.inf)
            log_out = torch.logsumexp(outside, -1, keepdim=True)
            share = log_p[:, -1:].exp()
            both = torch.cat([log_q[rows, index], log_out], -1)
            loss = torch.where(log_p > -math.inf, log_p.exp() * (log_p - both), torch.zeros_like(both)).sum(-1)
            wanted = torch.where(listed_too | (share == 0), torch.zeros_like(outside), (outside - log_out).exp() * share)
        wanted[rows, index] = log_p[:, :case["k"]].exp()
        keep = mask[part]
        losses.append(torch.where(keep, loss * temperature ** 2, torch.zeros_like(loss)))
        if case["gradient"]:
            grads.append((log_q.exp() - wanted) * temperature * keep[:, None])
    loss = torch.cat(losses)
    if not case["gradient"]:
        return [loss.reshape(case["rows"], *_space(case))]
    count = mask.sum()
    return [loss.sum() / count, _shaped(torch.cat(grads).div_(count), case)]


def _exact_verify(case, state):
    tokens, target, draft = state["tokens"], state["target"], state["draft"]
    rows, drafts = tokens.shape
    steps = target.shape[1]
    device = tokens.device
    length = torch.full((rows,), drafts, device=device) if state["lengths"] is None else state["lengths"].clone()
    alive = torch.ones(rows, dtype=torch.bool, device=device)
    accepted = torch.zeros(rows, dtype=torch.int64, device=device)
    answer = torch.full((rows, steps), -1, dtype=torch.int64, device=device)
    for t in range(steps):
        weight = target[:, t].double()
        drafted = alive & (t < length)
        if t < drafts:
            token = tokens[:, t]
            q = torch.ones_like(weight) if draft is None else draft[:, t].double()
            p = weight.gather(1, token[:, None])[:, 0]
            takes = drafted & (state["accept"][:, t].double() * q.gather(1, token[:, None])[:, 0] < p)
            if draft is None:
                excess = weight.scatter(1, token[:, None], 0.0)
            else:
                excess = torch.relu(weight - q)
            weight = torch.where((drafted & (excess.sum(1) > 0))[:, None], excess, weight)
        else:
            takes = torch.zeros_like(alive)
        draws = alive & ~takes
        total = weight.cumsum(1)
        found = torch.searchsorted(total, (state["sample"].double() * total[:, -1])[:, None], right=True)[:, 0]
        most = (weight > 0).double().mul_(torch.arange(1, case["classes"] + 1, device=device)).argmax(1)
        found = torch.minimum(found, most)
        answer[:, t] = torch.where(takes, token if t < drafts else found, torch.where(draws, found, answer[:, t]))
        accepted += takes
        alive = takes
    return [answer, accepted]
