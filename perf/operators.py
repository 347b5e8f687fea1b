"""The token operators of torchbiggraph_b200 as measurable cases: looking rows of a table up and the gradient of that, log
probabilities over rows of scores and their gradient, log probabilities over all rows of a table and their gradient.

  kind "lookup"         rows of a table by id, scaled
  kind "lookup_grad"    the dense gradient of the table: the rows' gradients summed by id
  kind "logprobs"       per row of scores: log probability of the target, entropy, log of the sum, rank, the best alternatives
  kind "logprobs_grad"  gradient of log probability and entropy with respect to the scores
  kind "table"          log probability and entropy of targets under queries . table^T, the scores never asked for
  kind "table_grad"     gradients of both with respect to the queries and the table

With `own` false every kind runs in its plain form: elementary torch operations in 32 bits, rounded once at the end.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
IGNORE = -100
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _package():
    place = os.path.join(os.getcwd(), "pytorch-biggraph_b200")
    if place not in sys.path:
        sys.path.insert(0, place)
    import torchbiggraph_b200
    return torchbiggraph_b200


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of five requests: the rows of their last tokens; latency
        dict(name="lookup_step", kind="lookup", n=5, rows=131_072, dim=4096, type="bf16", scale=64.0),
        # the tokens of a training batch in a table of this framework's own type and width
        dict(name="lookup_batch", kind="lookup", n=16_384, rows=100_003, dim=1024, type="fp32", scale=32.0),
        # the same batch's gradient: a few ids make up much of it, most rows of the table get none
        dict(name="lookup_grad_batch", kind="lookup_grad", n=16_384, rows=131_072, dim=2048, type="bf16", scale=math.sqrt(2048.0)),
        # both endpoints of 5000 edges over the 14,951 entities of the multi-relation graph; small enough for latency to count
        dict(name="lookup_grad_graph", kind="lookup_grad", n=10_000, rows=14_951, dim=400, type="fp32", scale=1.0),
        # a decoding step of four requests with twenty alternatives each: few long rows
        dict(name="logprobs_step", kind="logprobs", n=4, rows=131_072, pad=0, type="bf16", scale=1.25, top=20),
        # scoring what was sampled: an odd number of rows, entropy and eight alternatives
        dict(name="logprobs_batch", kind="logprobs", n=4099, rows=131_072, pad=0, type="bf16", scale=1.0, top=8),
        # the gradient of a policy's log probabilities and entropy over the same vocabulary
        dict(name="logprobs_grad_batch", kind="logprobs_grad", n=4096, rows=131_072, pad=0, type="bf16", scale=1.0, entropy=True),
        # rows of an odd number of half-precision scores: every row starts at another alignment
        dict(name="logprobs_grad_odd", kind="logprobs_grad", n=1000, rows=14_951, pad=0, type="fp16", scale=1.0, entropy=False),
        # seven hidden states against the whole table: the table is read once
        dict(name="table_step", kind="table", n=7, rows=131_072, dim=2048, type="bf16", scale=1.0),
        # 1000 queries of the multi-relation graph against all of its entities, in the tables' own type
        dict(name="table_batch", kind="table", n=1000, rows=14_951, dim=400, type="fp32", scale=1.0),
        # a training batch's loss against the whole table: the largest, on the tensor cores
        dict(name="table_grad_batch", kind="table_grad", n=4099, rows=65_536, dim=2048, type="bf16", scale=1.0, entropy=False),
        # the multi-relation graph's batch of 5000 edges trained against all entities, in the tables' own type
        dict(name="table_grad_graph", kind="table_grad", n=5000, rows=14_951, dim=400, type="fp32", scale=1.0, entropy=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "lookup_grad", "logprobs", "logprobs_grad", "table", "table_grad"])
    case = dict(kind=kind, type=rng.choice(["bf16", "fp32", "fp16"]), scale=rng.choice([1.0, 0.7, 2.5]))
    if kind in ("lookup", "lookup_grad"):
        case.update(n=_spread(rng, 1, 65_536), rows=_spread(rng, 500, 131_072), dim=_spread(rng, 30, 2048))
        if rng.random() < 0.5:
            case["dim"] = (case["dim"] + 31) // 32 * 32
    elif kind in ("logprobs", "logprobs_grad"):
        case.update(n=_spread(rng, 1, 4096), rows=_spread(rng, 300, 131_072), pad=rng.choice([0, 0, 24, 57]))
        if kind == "logprobs":
            case["top"] = rng.choice([0, 1, 5, 20, 32])
        else:
            case["entropy"] = rng.random() < 0.5
    else:
        case.update(n=_spread(rng, 1, 4096), rows=_spread(rng, 300, 65_536), dim=_spread(rng, 30, 2048))
        if rng.random() < 0.5:
            case["dim"] = (case["dim"] + 63) // 64 * 64
        if kind == "table_grad":
            case["entropy"] = rng.random() < 0.5
    return case


def work(case):
    """Every input once, every output once.  Of a looked-up table at most the rows asked for."""
    n, v, e = case["n"], case["rows"], BYTES[case["type"]]
    kind = case["kind"]
    if kind == "lookup":
        return {"bytes": 8 * n + (n + min(n, v)) * case["dim"] * e, "flops": n * case["dim"]}
    if kind == "lookup_grad":
        return {"bytes": 8 * n + (n + v) * case["dim"] * e, "flops": n * case["dim"]}
    if kind == "logprobs":
        return {"bytes": n * v * e + n * (8 + 20 + 12 * case["top"]), "flops": 6 * n * v}
    if kind == "logprobs_grad":
        return {"bytes": 2 * n * v * e + n * 24, "flops": 6 * n * v}
    d = case["dim"]
    if kind == "table":
        return {"bytes": (n + v) * d * e + n * 20, "flops": 2 * n * v * d}
    return {"bytes": 2 * (n + v) * d * e + n * 24, "flops": 6 * n * v * d}


# ----------------------------------------------------------------------------------------------- inputs
def _ids(n, rows, gen):
    """Ids whose frequency falls with the inverse of their rank, over permuted ids: a few make up much of a batch."""
    rank = torch.exp(torch.rand(n, device=DEVICE, generator=gen, dtype=torch.float64) * math.log(rows + 1.0)).long() - 1
    return torch.randperm(rows, device=DEVICE, generator=gen)[rank.clamp_(0, rows - 1)]


def _targets(n, rows, gen):
    """One in thirty-two is padding."""
    t = _ids(n, rows, gen)
    return torch.where(torch.rand(n, device=DEVICE, generator=gen) < 1 / 32, torch.full_like(t, IGNORE), t)


def _statistics(z):
    """Log of the sum and entropy of rows of scores, for the gradients' inputs; a slab of rows at a time."""
    lse, ent = [], []
    for part in z.split(256):
        x = part.float()
        m = x.amax(1, keepdim=True)
        d = x - m
        e = torch.exp(d)
        s = e.sum(1, keepdim=True)
        lse.append((m + torch.log(s)).squeeze(1))
        ent.append((torch.log(s) - torch.where(e > 0, d * e, 0.0).sum(1, keepdim=True) / s).squeeze(1))
    return torch.cat(lse), torch.cat(ent)


def _row_gradients(case, randn):
    """Of a mean over the rows; half precision comes with a loss scale of the number of rows."""
    size = 1.0 if case["type"] == "fp16" else 1.0 / case["n"]
    g = randn(case["n"]).mul_(size)
    return g, randn(case["n"]).mul_(0.1 * size) if case["entropy"] else None


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, n, rows, dtype = case["kind"], case["n"], case["rows"], TYPES[case["type"]]
    randn = lambda *shape: torch.randn(*shape, device=DEVICE, generator=gen)  # noqa: E731
    s = dict(case)
    if kind == "lookup":
        s["table"] = randn(rows, case["dim"]).mul_(0.02).to(dtype)
        s["ids"] = _ids(n, rows, gen)
    elif kind == "lookup_grad":
        s["ids"] = _ids(n, rows, gen)
        s["grad"] = randn(n, case["dim"]).mul_(0.01).to(dtype)
    elif kind in ("logprobs", "logprobs_grad"):
        # rows of scores with room behind them, as where a vocabulary is padded; the last 1 % of the ids is never allowed
        x = randn(n, rows + case["pad"]).mul_(2.0)
        s["targets"] = _targets(n, rows, gen)
        at = s["targets"].clamp(min=0).unsqueeze(1)
        x.scatter_add_(1, at, randn(n, 1).add_(6.0))
        banned = torch.arange(rows + case["pad"], device=DEVICE) >= rows - rows // 100
        x.masked_fill_(banned & (torch.arange(rows + case["pad"], device=DEVICE) != at), -math.inf)
        s["logits"] = x.to(dtype)[:, :rows]
        del x
        if kind == "logprobs_grad":
            s["lse"], s["entropy_of"] = _statistics(s["logits"] if case["scale"] == 1.0 else s["logits"].float() * case["scale"])
            s["g"], s["h"] = _row_gradients(case, randn)
    else:
        d = case["dim"]
        s["table"] = (randn(rows, d) / math.sqrt(d)).to(dtype)
        s["targets"] = _targets(n, rows, gen)
        # queries that lean towards their targets, as in the middle of a training run: scores of a spread of two
        s["queries"] = (randn(n, d).mul_(2.0) + 4.0 * s["table"][s["targets"].clamp(min=0)].float()).to(dtype)
        if kind == "table_grad":
            lse, ent = [], []
            t = s["table"].float()
            for q in s["queries"].split(1024):
                a, b = _statistics((q.float() @ t.T) * case["scale"])
                lse.append(a)
                ent.append(b)
            s["lse"], s["entropy_of"] = torch.cat(lse), torch.cat(ent)
            s["g"], s["h"] = _row_gradients(case, randn)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_lookup(s):
    return {"rows": (s["table"][s["ids"]].float() * s["scale"]).to(s["table"].dtype)}


def _plain_lookup_grad(s):
    out = torch.zeros(s["rows"], s["dim"], device=DEVICE)
    out.index_add_(0, s["ids"], s["grad"].float())
    return {"grad": (out * s["scale"]).to(s["grad"].dtype)}


def _plain_statistics(z, targets):
    real = targets >= 0
    at = targets.clamp(min=0).unsqueeze(1)
    m = z.amax(1, keepdim=True)
    d = z - m
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    # (-inf) * 0 is 0 here
    entropy = log_total - torch.where(e > 0, d * e, 0.0).sum(1) / total
    logprob = d.gather(1, at).squeeze(1) - log_total
    zero = torch.zeros_like(logprob)
    return torch.where(real, logprob, zero), torch.where(real, entropy, zero), torch.where(real, m.squeeze(1) + log_total, zero)


def _plain_logprobs(s):
    x, targets, top = s["logits"].float(), s["targets"], s["top"]
    logprob, entropy, lse = _plain_statistics(x * s["scale"], targets)
    real = targets >= 0
    at = targets.clamp(min=0).unsqueeze(1)
    mine = x.gather(1, at)
    index = torch.arange(s["rows"], device=DEVICE)
    rank = 1 + ((x > mine) | ((x == mine) & (index < at))).sum(1)
    out = dict(logprob=logprob, entropy=entropy, lse=lse, rank=torch.where(real, rank, 0))
    if top:
        # whole numbers in the order of the scores, equal scores in the order of falling index
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32 + (2 ** 31 - index)
        ids = 2 ** 31 - (torch.topk(order, top, dim=1).values & 0xFFFFFFFF)
        best = x.gather(1, ids) * s["scale"] - lse.unsqueeze(1)
        out["top_ids"] = torch.where(real.unsqueeze(1), ids, -1)
        out["top_logprobs"] = torch.where(real.unsqueeze(1), best, 0.0)
    return out


def _plain_score_grad(z, s):
    """Gradient with respect to rows of scaled scores."""
    targets = s["targets"]
    real = targets >= 0
    g = torch.where(real, s["g"], 0.0).unsqueeze(1)
    logp = z - s["lse"].unsqueeze(1)
    p = torch.exp(logp)
    dz = -g * p
    if s["h"] is not None:
        h = torch.where(real, s["h"], 0.0).unsqueeze(1)
        dz = dz - torch.where(p > 0, h * p * (logp + s["entropy_of"].unsqueeze(1)), 0.0)
    return dz.scatter_add(1, targets.clamp(min=0).unsqueeze(1), g)


def _plain_logprobs_grad(s):
    return {"grad": (s["scale"] * _plain_score_grad(s["logits"].float() * s["scale"], s)).to(s["logits"].dtype)}


def _plain_table(s):
    z = (s["queries"].float() @ s["table"].float().T) * s["scale"]
    logprob, entropy, lse = _plain_statistics(z, s["targets"])
    return dict(logprob=logprob, entropy=entropy, lse=lse)


def _plain_table_grad(s):
    q, t = s["queries"].float(), s["table"].float()
    dz = s["scale"] * _plain_score_grad((q @ t.T) * s["scale"], s)
    return dict(queries=(dz @ t).to(s["queries"].dtype), table=(dz.T @ q).to(s["table"].dtype))


_PLAIN = {"lookup": _plain_lookup, "lookup_grad": _plain_lookup_grad, "logprobs": _plain_logprobs,
          "logprobs_grad": _plain_logprobs_grad, "table": _plain_table, "table_grad": _plain_table_grad}


def _own_run(s):
    T = _package()
    kind, scale = s["kind"], s["scale"]
    if kind == "lookup":
        return {"rows": T.embedding_lookup(s["table"], s["ids"], scale=scale)}
    if kind == "lookup_grad":
        return {"grad": T.embedding_lookup_grad(s["grad"], s["ids"], s["rows"], scale=scale)}
    if kind == "logprobs":
        r = T.token_logprobs(s["logits"], s["targets"], scale=scale, top=s["top"])
        out = dict(logprob=r.logprob, entropy=r.entropy, lse=r.lse, rank=r.rank)
        if s["top"]:
            out.update(top_ids=r.top_ids, top_logprobs=r.top_logprobs)
        return out
    if kind == "logprobs_grad":
        return {"grad": T.token_logprobs_grad(s["logits"], s["targets"], s["lse"], s["entropy_of"], s["g"], s["h"], scale=scale)}
    if kind == "table":
        r = T.table_logprobs(s["queries"], s["table"], s["targets"], scale=scale)
        return dict(logprob=r.logprob, entropy=r.entropy, lse=r.lse)
    dq, dt = T.table_logprobs_grad(s["queries"], s["table"], s["targets"], s["lse"], s["entropy_of"], s["g"], s["h"], scale=scale)
    return dict(queries=dq, table=dt)


def run(state):
    return _own_run(state) if own else _PLAIN[state["kind"]](state)


# ------------------------------------------------------------------------------- the definition, 64 bits
def _exact_rows(z, targets, scale):
    """Log-softmax of slabs of rows from torch's 64-bit logsumexp."""
    z = z.double() * scale
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    entropy = torch.special.entr(logp.exp()).sum(1)
    padding = targets == IGNORE
    logprob = logp[torch.arange(len(z), device=z.device), targets.clamp(min=0)]
    return tuple(x.masked_fill(padding, 0.0) for x in (logprob, entropy, lse)) + (logp,)


def _exact_weights(logp, s, part):
    """d(sum of g logprob + h entropy) / d(score) of slab `part` from its log probabilities."""
    keep = (s["targets"][part] != IGNORE).double()
    p = logp.exp()
    w = torch.zeros_like(p)
    w[torch.arange(len(p), device=p.device), s["targets"][part].clamp(min=0)] = 1.0
    w = (s["g"][part].double() * keep)[:, None] * (w - p)
    if s["h"] is not None:
        w += (s["h"][part].double() * keep)[:, None] * (torch.special.entr(p) - p * s["entropy_of"][part].double()[:, None])
    return w * s["scale"]


def exact(case, seed):
    s = prepare(case, seed)
    kind, n = case["kind"], case["n"]
    slabs = [slice(i, min(i + 512, n)) for i in range(0, n, 512)]
    if kind == "lookup":
        return {"rows": s["table"].double().index_select(0, s["ids"]) * s["scale"]}
    if kind == "lookup_grad":
        order = torch.sort(s["ids"], stable=True)
        ids, count = torch.unique_consecutive(order.values, return_counts=True)
        out = torch.zeros(case["rows"], case["dim"], device=DEVICE, dtype=torch.float64)
        out[ids] = torch.segment_reduce(s["grad"].double()[order.indices] * s["scale"], "sum", lengths=count)
        return {"grad": out}
    if kind == "logprobs":
        got = [[], [], [], []]
        for part in slabs:
            logprob, entropy, lse, logp = _exact_rows(s["logits"][part], s["targets"][part], s["scale"])
            best = logp.topk(case["top"], dim=1).values if case["top"] else logp[:, :0]
            for to, x in zip(got, (logprob, entropy, lse, best.masked_fill((s["targets"][part] == IGNORE)[:, None], 0.0))):
                to.append(x)
        logprob, entropy, lse, best = map(torch.cat, got)
        out = dict(logprob=logprob, entropy=entropy, lse=lse, rank=None)
        if case["top"]:
            out.update(top_ids=None, top_logprobs=best)
        return out
    if kind == "logprobs_grad":
        return {"grad": torch.cat([_exact_weights(s["logits"][p].double() * s["scale"] - s["lse"][p].double()[:, None], s, p) for p in slabs])}
    t = s["table"].double()
    if kind == "table":
        got = [_exact_rows(s["queries"][p].double() @ t.T, s["targets"][p], s["scale"])[:3] for p in slabs]
        return dict(zip(("logprob", "entropy", "lse"), map(torch.cat, zip(*got))))
    dq, dt = [], torch.zeros_like(t)
    for p in slabs:
        q = s["queries"][p].double()
        w = _exact_weights((q @ t.T) * s["scale"] - s["lse"][p].double()[:, None], s, p)
        dq.append(w @ t)
        dt += w.T @ q
    return dict(queries=torch.cat(dq), table=dt)
