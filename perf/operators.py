"""The losses over the tied output table, as cases to measure.

Cross entropy over the whole vocabulary and distillation from a teacher's top
logits, both on hidden rows and the embedding table of the output head, each
forward alone (scores of given tokens) and as the loss part of a training step
(forward, then both gradients).
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
IGNORED = -1  # int32 view of the invalid token id: a row without a target


def listed():
    return [
        # log-probability of one token: the smallest call, the table read once
        dict(name="xent forward 1", op="xent", train=False, rows=1, vocab=49152, hidden=576,
             dtype="f16", ignored=0.0),
        # a decode batch of 64 sequences scored
        dict(name="xent forward 64", op="xent", train=False, rows=64, vocab=49152, hidden=576,
             dtype="bf16", ignored=0.0),
        # evaluation of one sequence of 1,024 positions
        dict(name="xent forward 1024", op="xent", train=False, rows=1024, vocab=49152, hidden=576,
             dtype="f16", ignored=0.1),
        # a training step on a short sequence
        dict(name="xent train 256", op="xent", train=True, rows=256, vocab=49152, hidden=576,
             dtype="f16", ignored=0.1),
        # odd sizes everywhere, a width that ends inside a 64-wide chunk
        dict(name="xent train 1001 odd", op="xent", train=True, rows=1001, vocab=32003, hidden=328,
             dtype="bf16", ignored=0.3),
        # a whole training batch of eight sequences: the largest
        dict(name="xent train 8192", op="xent", train=True, rows=8192, vocab=49152, hidden=576,
             dtype="f16", ignored=0.05),
        # divergence from the teacher, decode batch
        dict(name="distill forward 48", op="distill", train=False, rows=48, vocab=49152, hidden=576,
             dtype="f16", most=32, temperature=1.0, empty=0.05),
        # evaluation against a wide teacher set
        dict(name="distill forward 2000", op="distill", train=False, rows=2000, vocab=49152,
             hidden=576, dtype="bf16", most=256, temperature=2.0, empty=0.05),
        # a small vocabulary and a narrow student
        dict(name="distill train 333 odd", op="distill", train=True, rows=333, vocab=8191,
             hidden=192, dtype="f16", most=17, temperature=1.5, empty=0.2),
        # a training step from a stored teacher
        dict(name="distill train 4096", op="distill", train=True, rows=4096, vocab=49152,
             hidden=576, dtype="bf16", most=64, temperature=2.0, empty=0.05),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = 8192 * 49152 * 576
    while True:
        case = dict(op=rng.choice(("xent", "distill")), train=rng.random() < 0.6,
                    rows=_log_uniform(rng, 1, 8192), vocab=_log_uniform(rng, 1000, 50000),
                    hidden=8 * _log_uniform(rng, 8, 128), dtype=rng.choice(("f16", "bf16")))
        if case["op"] == "xent":
            case["ignored"] = rng.choice((0.0, 0.1, 0.5))
        else:
            case.update(most=_log_uniform(rng, 1, 300), empty=rng.choice((0.0, 0.1)),
                        temperature=rng.choice((1.0, 1.5, 4.0)))
        if case["rows"] * case["vocab"] * case["hidden"] <= most:
            return case


def prepare(case, seed):
    """Normed hidden rows that lean towards a target by different amounts, the
    table, targets or teacher sets in CSR form, and the gradient of the losses
    (their mean, token weights and a loss scale for fp16)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, width = case["rows"], case["vocab"], case["hidden"]
    dtype = _TYPES[case["dtype"]]

    def rand(*size):
        return torch.rand(*size, generator=gen, device="cuda")

    table = (0.02 * torch.randn(vocab, width, generator=gen, device="cuda")).to(dtype)
    # frequent tokens have low ids
    targets = (vocab * rand(rows) ** 2).long().clamp_(max=vocab - 1)
    x = torch.randn(rows, width, generator=gen, device="cuda")
    x = x + 2.5 * rand(rows, 1) * table[targets].float() / 0.02
    hidden = (x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-5)).to(dtype)
    scale = 1024.0 if case["dtype"] == "f16" else 1.0
    state = {"op": case["op"], "train": case["train"], "hidden": hidden, "table": table,
             "grad": (0.5 + rand(rows)) * (scale / rows), "own": {}}
    if case["op"] == "xent":
        state["targets"] = torch.where(rand(rows) < case["ignored"], IGNORED, targets).int()
    else:
        most = min(case["most"], vocab)
        # the target and other likely tokens, ascending; repeated ones fall out
        ids = (vocab * rand(rows, most) ** 2).long().clamp_(max=vocab - 1)
        ids[:, 0] = targets
        ids = ids.sort(1).values
        keep = torch.ones_like(ids, dtype=torch.bool)
        keep[:, 1:] = ids[:, 1:] != ids[:, :-1]
        keep &= (rand(rows, most) < 0.9) | (ids == targets[:, None])
        keep &= rand(rows, 1) >= case["empty"]
        logits = 3.0 * torch.randn(rows, most, generator=gen, device="cuda")
        logits += 6.0 * (ids == targets[:, None])
        # some stored entries are masked out
        logits = torch.where((rand(rows, most) < 0.02) & (ids != targets[:, None]), -math.inf,
                             logits)
        state["offsets"] = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
        state["offsets"][1:] = keep.sum(1).cumsum(0)
        state["ids"] = ids[keep].int()
        state["logits"] = logits[keep]
        state["temperature"] = case["temperature"]
    state["stream"] = torch.cuda.Stream()
    state["stream"].wait_stream(torch.cuda.current_stream())
    return state


def run(state):
    with torch.cuda.stream(state["stream"]):
        if own:
            return _run_own(state)
        return _run_plain(state)


def _run_own(s):
    from market_sim_b200 import head

    keep = s["own"]  # the workspaces and output buffers a program keeps from step to step
    if not keep:
        keep["loss"] = head.DenseLoss(s["table"], s["hidden"].shape[0], stream=s["stream"],
                                      backward=s["train"])
        keep["losses"] = torch.empty_like(s["grad"])
        keep["lse"] = torch.empty_like(s["grad"])
        if s["train"]:
            keep["d_hidden"] = torch.empty_like(s["hidden"])
            keep["d_table"] = torch.empty_like(s["table"])
    loss = keep["loss"]
    if s["op"] == "xent":
        given = (s["hidden"], s["targets"])
        losses, lse = loss.cross_entropy(*given, losses=keep["losses"], lse=keep["lse"])
        if s["train"]:
            d_hidden, d_table = loss.cross_entropy_backward(
                *given, lse, s["grad"], d_hidden=keep["d_hidden"], d_embedding=keep["d_table"])
    else:
        given = (s["hidden"], s["offsets"], s["ids"], s["logits"], s["temperature"])
        losses, lse = loss.distill(*given, losses=keep["losses"], lse=keep["lse"])
        if s["train"]:
            d_hidden, d_table = loss.distill_backward(
                *given, lse, s["grad"], d_hidden=keep["d_hidden"], d_embedding=keep["d_table"])
    if not s["train"]:
        return {"losses": losses, "lse": lse}
    return {"losses": losses, "lse": lse, "d_hidden": d_hidden, "d_table": d_table}


def _run_plain(s):
    hidden, table = s["hidden"].float(), s["table"].float()
    rows = hidden.shape[0]
    scores = hidden @ table.T
    if s["op"] == "xent":
        temperature, gain = 1.0, 1.0
        active = s["targets"] >= 0
        at_row = torch.nonzero(active)[:, 0]
        at_id = s["targets"][at_row].long()
        q = torch.ones_like(at_row, dtype=torch.float32)
        entropy = torch.zeros_like(q)
    else:
        temperature = s["temperature"]
        gain = temperature * temperature
        lengths = (s["offsets"][1:] - s["offsets"][:-1]).long()
        at_row = torch.repeat_interleave(torch.arange(rows, device=hidden.device), lengths)
        at_id = s["ids"].long()
        t = s["logits"] / temperature
        top = torch.full((rows,), -math.inf, device=hidden.device)
        top = top.scatter_reduce(0, at_row, t, "amax")
        active = top > -math.inf
        e = torch.where(active[at_row], torch.exp(t - top[at_row]), torch.zeros_like(t))
        total = torch.zeros(rows, device=hidden.device).index_add_(0, at_row, e)
        q = torch.where(active[at_row], e / total[at_row], torch.zeros_like(t))
        log_q = t - top[at_row] - torch.log(total[at_row])
        entropy = torch.where(q > 0, q * log_q, torch.zeros_like(q))
        scores = scores / temperature
    top = scores.amax(1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    terms = entropy + q * (lse[at_row] - scores[at_row, at_id])
    losses = gain * torch.zeros(rows, device=hidden.device).index_add_(0, at_row, terms)
    if not s["train"]:
        return {"losses": losses, "lse": lse}
    p = p / total
    p.index_put_((at_row, at_id), -q, accumulate=True)
    p = p * torch.where(active, s["grad"] * (gain / temperature), torch.zeros_like(lse))[:, None]
    return {"losses": losses, "lse": lse, "d_hidden": (p @ table).to(s["hidden"].dtype),
            "d_table": (p.T @ hidden).to(s["table"].dtype)}


def _active_rows(case):
    return max(1.0, case["rows"] * (1.0 - case.get("ignored", case.get("empty"))))


def work(case):
    """Inputs read once, outputs written once; one product forward, two more
    for the gradients, on the rows that have a target."""
    rows, vocab, width = case["rows"], case["vocab"], case["hidden"]
    entries = rows if case["op"] == "xent" else rows * min(case["most"], vocab)
    size = 2 * (rows + vocab) * width + 8 * rows + 8 * entries
    flops = 2.0 * _active_rows(case) * vocab * width
    if case["train"]:
        size += 2 * (rows + vocab) * width + 4 * rows
        flops *= 3
    return {"bytes": size, "flops": flops}


def exact(case, seed):
    """The definitions in 64 bits, 512 rows at a time: dense teacher
    distributions and log_softmax."""
    s = prepare(case, seed)
    torch.cuda.synchronize()
    hidden, table = s["hidden"].double(), s["table"].double()
    rows, vocab = hidden.shape[0], table.shape[0]
    grad = s["grad"].double()
    temperature = s.get("temperature", 1.0)
    losses, lse, d_hidden = [], [], []
    d_table = torch.zeros_like(table)
    for r0 in range(0, rows, 512):
        r1 = min(rows, r0 + 512)
        wanted = torch.zeros(r1 - r0, vocab, dtype=torch.float64, device="cuda")
        if case["op"] == "xent":
            t = s["targets"][r0:r1].long()
            has = t >= 0
            wanted[torch.arange(r1 - r0, device="cuda")[has], t[has]] = 1.0
        else:
            off = s["offsets"].tolist()
            teacher = torch.full_like(wanted, -math.inf)
            lengths = torch.tensor([off[r + 1] - off[r] for r in range(r0, r1)], device="cuda")
            where = torch.repeat_interleave(torch.arange(r1 - r0, device="cuda"), lengths)
            part = slice(off[r0], off[r1])
            teacher[where, s["ids"][part].long()] = s["logits"][part].double()
            has = torch.isfinite(teacher).any(1)
            wanted[has] = torch.softmax(teacher[has] / temperature, 1)
        scores = (hidden[r0:r1] @ table.T) / temperature
        log_p = torch.log_softmax(scores, 1)
        lse.append((scores - log_p)[:, 0])
        terms = torch.special.xlogy(wanted, wanted) - wanted * log_p
        losses.append(temperature ** 2 * terms.sum(1))
        if case["train"]:
            d = temperature * (log_p.exp() - wanted) * (grad[r0:r1] * has)[:, None]
            d_hidden.append(d @ table)
            d_table += d.T @ hidden[r0:r1]
    out = {"losses": torch.cat(losses), "lse": torch.cat(lse)}
    if case["train"]:
        out.update(d_hidden=torch.cat(d_hidden), d_table=d_table)
    return out
