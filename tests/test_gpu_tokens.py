"""The token operators against their definitions in 64 bits: rows by id and their gradient, log probabilities over rows of scores
and their gradient.

Tolerances: a result is rounded to its type once, by at most half a step, finfo.eps / 2 of its value.  What comes before is fp32:
  - a sum of c terms is off by at most (c - 1) 2^-24 of the sum of the terms' sizes;
  - log probabilities, entropy and lse: an exponential 2^y, |y| <= 150 where it counts, with y off by 3 roundings and ex2 by 2 ulp, is
    relatively off by at most 150 * 3 * 2^-24 + 2^-22 < 3e-5, which only scores 100 below the largest reach; those within 20 of it,
    which make up the sums, stay below 6e-6.  S and T carry that and the sums' own roundings, thread by thread and joined
    (below 600 terms each and a tree of 11: 4e-5 at the worst of all signs, a hundredth of that in the mean); 2e-5 is used, relative to
    1 + |lse| (the larger of what is subtracted) resp. 1 + |entropy| + log S."""
import math

import pytest
import torch

import torchbiggraph_b200 as T

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def f32(scale):
    """A scale as the entry points take it, in single precision: 1.3 is another number there."""
    return float(torch.tensor(scale, dtype=torch.float32))


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, rel, scale, floor=0.0):
    """|got - want| <= rel * scale + floor everywhere, NaN and infinities in the same places."""
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    ok = want.isfinite()
    err = ((got - want).abs() - (rel * (scale if torch.is_tensor(scale) else torch.full_like(want, scale)) + floor))[ok]
    assert err.numel() == 0 or err.max().item() <= 0, err.max().item()


# ------------------------------------------------------------------------------------------------ lookup
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (3, 7, 2), (5, 100, 37), (64, 50, 100), (33, 1000, 400), (700, 300, 1026), (9, 10, 4096), (2, 3, 65_536),
                                        (3000, 5000, 256)])
def test_lookup(dtype, n, rows, dim):
    g = gen(n + dim)
    table = torch.randn(rows, dim, device=DEV, generator=g).to(dtype)
    ids = torch.randint(0, rows, (n,), device=DEV, generator=g)
    close(T.embedding_lookup(table, ids, scale=1.7), table.double()[ids] * 1.7, half_step(dtype) + 2 ** -23, (table.double()[ids] * 1.7).abs(),
          floor=torch.finfo(dtype).smallest_normal)
    assert torch.equal(T.embedding_lookup(table, ids), table[ids])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("stride,first", [(40, 0), (41, 0), (40, 1), (48, 3)])
def test_lookup_of_a_strided_table(dtype, stride, first):
    g = gen(stride)
    table = torch.randn(50, stride, device=DEV, generator=g).to(dtype)[:, first:first + 36]
    ids = torch.randint(0, 50, (4, 5), device=DEV, generator=g)
    got = T.embedding_lookup(table, ids)
    assert got.shape == (4, 5, 36) and torch.equal(got, table[ids])
    assert torch.equal(T.embedding_lookup(table, ids.t()), table[ids.t()])
    assert T.embedding_lookup(table, ids[:0]).shape == (0, 5, 36)


def test_lookup_reports_ids_outside_of_the_table():
    table = torch.randn(10, 8, device=DEV)
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = T.embedding_lookup(table, torch.tensor([3, -1, 10, 2 ** 40, 0], device=DEV), errors=errors)
    assert torch.equal(got[[0, 4]], table[[3, 0]]) and got[1:4].isnan().all()
    with pytest.raises(IndexError):
        T.check_errors(errors)
    T.check_errors(errors)
    assert T.embedding_lookup(table, torch.tensor([11], device=DEV)).isnan().all()          # (without an error word as well)


def _grad_want(grad, ids, rows, scale):
    out = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device=DEV)
    ok = (ids >= 0) & (ids < rows)
    out.index_add_(0, ids[ok], grad.double()[ok])
    size = torch.zeros_like(out).index_add_(0, ids[ok], grad.double()[ok].abs())
    return out * scale, size * abs(scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim,kind", [(1, 1, 1, "any"), (1, 500, 33, "any"), (16, 4, 8, "any"), (17, 4, 8, "one"), (33, 3, 100, "few"), (1000, 7, 400, "few"),
                                             (4096, 3000, 130, "any"), (5000, 2000, 1, "one"), (2500, 100_003, 24, "few"), (20_001, 4000, 64, "any"),
                                             (300_000, 1000, 4, "any"), (263_000, 70_000, 8, "one"), (512, 700, 2048, "few"), (511, 3, 200, "any"),
                                             (513, 40, 96, "few"), (300, 9000, 1, "any"), (512, 1, 516, "one"), (1536, 700, 516, "few"), (1536, 9, 33, "one"),
                                             (1537, 700, 130, "few"), (900, 5, 2048, "any"), (1535, 20_000, 1026, "any"), (9, 2, 1024, "one")])
def test_lookup_grad(dtype, n, rows, dim, kind):
    g = gen(n + dim)
    ids = torch.randint(0, rows, (n,), device=DEV, generator=g)
    if kind == "one":
        ids.fill_(rows - 1)
    elif kind == "few":
        ids = torch.where(torch.rand(n, device=DEV, generator=g) < 0.8, ids % 3 % rows, ids)
    grad = torch.randn(n, dim, device=DEV, generator=g).to(dtype)
    want, size = _grad_want(grad, ids, rows, 0.5)
    most = int(torch.bincount(ids).max())
    rel = (most + 4) * 2 ** -24
    got = T.embedding_lookup_grad(grad, ids, rows, scale=0.5)
    close(got, want, 1.0, half_step(dtype) * want.abs() + rel * size, floor=torch.finfo(dtype).smallest_normal)
    assert torch.equal(got, T.embedding_lookup_grad(grad, ids, rows, scale=0.5))             # the same bits again
    # added to what is there: rows without an id keep their bits
    base = torch.randn(rows, dim, device=DEV, generator=g).to(dtype)
    got = T.embedding_lookup_grad(grad, ids, rows, scale=0.5, out=base.clone(), accumulate=True)
    close(got, base.double() + want, 1.0, half_step(dtype) * (base.double() + want).abs() + rel * size + 2 ** -24 * base.double().abs(), floor=torch.finfo(dtype).smallest_normal)
    empty = torch.ones(rows, dtype=torch.bool, device=DEV)
    empty[ids] = False
    assert torch.equal(got[empty], base[empty])


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_grad_strides_and_bad_ids(dtype):
    g = gen(5)
    wide = torch.randn(40, 61, device=DEV, generator=g).to(dtype)
    for first, dim in ((0, 56), (1, 48), (3, 33)):
        grad = wide[:, first:first + dim]
        ids = torch.randint(0, 9, (40,), device=DEV, generator=g)
        ids[[3, 17, 39]] = torch.tensor([-5, 9, 2 ** 50], device=DEV)
        room = torch.full((9, 70), 7.0, device=DEV, dtype=dtype)
        errors = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = T.embedding_lookup_grad(grad, ids, 9, out=room[:, 2:2 + dim], errors=errors)
        want, size = _grad_want(grad, ids, 9, 1.0)
        close(out, want, 1.0, half_step(dtype) * want.abs() + 44 * 2 ** -24 * size)
        assert (room[:, :2] == 7).all() and (room[:, 2 + dim:] == 7).all() and errors.item() == 1
    assert (T.embedding_lookup_grad(wide[:0], torch.empty(0, dtype=torch.long, device=DEV), 4) == 0).all()
    one = T.embedding_lookup_grad(wide.view(8, 5, 61), torch.zeros(8, 5, dtype=torch.long, device=DEV), 1)
    assert one.shape == (1, 61)


def test_lookup_gradient_is_the_slope_of_the_lookup():
    """<W + d, .> differences: the lookup is linear in the table, so one step of any size gives the slope."""
    g = gen(1)
    ids = torch.randint(0, 30, (100,), device=DEV, generator=g)
    out_grad = torch.randn(100, 20, device=DEV, generator=g)
    W, d = torch.randn(30, 20, device=DEV, generator=g), torch.randn(30, 20, device=DEV, generator=g)
    dW = T.embedding_lookup_grad(out_grad, ids, 30, scale=3.0).double()
    slope = ((T.embedding_lookup(W + d, ids, scale=3.0).double() - T.embedding_lookup(W, ids, scale=3.0).double()) * out_grad.double()).sum()
    assert abs((dW * d.double()).sum() - slope).item() < 2000 * 20 * 2 ** -22


# --------------------------------------------------------------------------------------------- log probabilities
def _scores(n, vocab, dtype, seed, kind="plain", pad=0):
    g = gen(seed)
    x = torch.randn(n, vocab + pad, device=DEV, generator=g) * 3
    if kind == "ties":
        x = x.round()
    if kind == "sharp":
        x[torch.arange(n), torch.randint(0, vocab, (n,), device=DEV, generator=g)] += 30
    if kind == "masked":
        x[torch.rand(n, vocab + pad, device=DEV, generator=g) < 0.7] = -math.inf
        x[0] = -math.inf
        if n > 1:
            x[1] = torch.finfo(dtype).min
        if n > 2:
            x[2] = torch.finfo(dtype).min
            x[2, vocab // 2] = 1.0
        if n > 3:
            x[3, :-1] = -math.inf
    return x.to(dtype)[:, :vocab]


def _want(x, targets, scale, top):
    z = x.double() * f32(scale)
    m = z.amax(1)
    # (against the maximum first: next to a row of the type's lowest value, log 2 is lost in 64 bits too)
    d = z - torch.where(m == -math.inf, 0.0, m)[:, None]
    log_sum = torch.logsumexp(d, 1)
    lse, logp = m + torch.where(m == -math.inf, 0.0, log_sum), d - log_sum[:, None]
    logp[lse == -math.inf] = -math.inf
    ent = torch.special.entr(logp.exp()).sum(1)
    real = targets >= 0
    t = targets.clamp(min=0)[:, None]
    mine = x.gather(1, t)
    ids = torch.arange(x.shape[1], device=DEV)
    rank = 1 + ((x > mine) | ((x == mine) & (ids < t))).sum(1)
    order = torch.sort(torch.where(x.isnan(), -math.inf, x.float()), dim=1, descending=True, stable=True).indices[:, :top]
    z0 = lambda v, pad=0: torch.where(real if v.dim() == 1 else real[:, None], v, pad)  # noqa: E731
    return z0(logp.gather(1, t)[:, 0]), z0(ent), z0(lse), z0(rank), z0(logp.gather(1, order)), z0(order, -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["plain", "ties", "sharp", "masked"])
@pytest.mark.parametrize("n,vocab,pad,top", [(1, 1, 0, 1), (4, 2, 0, 2), (5, 31, 0, 31), (7, 33, 6, 32), (6, 1000, 0, 0), (9, 1025, 0, 5), (3, 14_951, 57, 20), (300, 2048, 0, 8),
                                             (2, 131_072, 0, 20), (1, 70_001, 3, 32), (700, 517, 0, 1)])
def test_logprobs(dtype, kind, n, vocab, pad, top):
    x = _scores(n, vocab, dtype, n + vocab, kind, pad)
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen(vocab))
    if n > 5:
        targets[5] = -100
    r = T.token_logprobs(x, targets, scale=0.8, top=top)
    logprob, ent, lse, rank, best, ids = _want(x, targets, 0.8, top)
    size = 1 + torch.where(lse.isfinite(), lse.abs(), 1.0)
    close(r.lse, lse, 2e-5, size)
    close(r.logprob, logprob, 2e-5, size + torch.where(logprob.isfinite(), logprob.abs(), 0.0))
    close(r.entropy, ent, 2e-5, 1 + ent + math.log(vocab))
    assert torch.equal(r.rank, rank)
    if top:
        assert torch.equal(r.top_ids, ids)
        close(r.top_logprobs, best, 2e-5, size[:, None] + torch.where(best.isfinite(), best.abs(), 0.0))
    else:
        assert r.top_ids is None and r.top_logprobs is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("base", [-1e30, -1e9, -65_000.0, -300.0, 3e4, 1e6, 1e30])
@pytest.mark.parametrize("n,vocab", [(3, 11), (2, 30_000), (700, 2051)])
def test_logprobs_far_from_zero(dtype, base, n, vocab):
    """Rows that a mask of -1e9 leaves nothing of, and others around a large number: the differences of the scores are exact, and so the
    log probabilities, which do not pass through lse, are as good as those around zero: 2e-5 of 1 + their size."""
    if dtype == torch.float16 and abs(base) > 65_504:
        base = math.copysign(6e4, base)
    x = torch.full((n, vocab), base, device=DEV).to(dtype)
    step = x[0, 0].float().abs().item() * torch.finfo(dtype).eps               # the next numbers of the type, where they are near
    if step < 64:
        x = (x.float() + torch.randint(-3, 4, (n, vocab), device=DEV, generator=gen(9)) * step).to(dtype)
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen(3))
    r = T.token_logprobs(x, targets, top=4)
    z = x.double() - x.double().amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1)
    logprob = z.gather(1, targets[:, None])[:, 0] - lse
    assert ((r.logprob.double() - logprob).abs() <= 2e-5 * (1 + logprob.abs())).all()
    p = torch.softmax(z, 1)
    ent = torch.special.entr(p).sum(1)
    assert ((r.entropy.double() - ent).abs() <= 2e-5 * (1 + ent + math.log(vocab))).all()
    best = z.gather(1, r.top_ids) - lse[:, None]
    assert ((r.top_logprobs.double() - best).abs() <= 2e-5 * (1 + best.abs())).all()
    top = x.double().amax(1)
    assert ((r.lse.double() - top - lse).abs() <= 2e-5 * (1 + lse.abs()) + 2 ** -23 * top.abs()).all()


def test_logprobs_of_rows_of_equal_scores_keep_the_order_of_ids():
    for vocab in (64, 5000, 131_073):
        for value in (0.0, -3.0, -math.inf):
            x = torch.full((3, vocab), value, device=DEV, dtype=torch.bfloat16)
            x[1, ::2] = -x[1, ::2] if value == 0.0 else x[1, ::2]              # -0 and 0 are equal
            r = T.token_logprobs(x, torch.tensor([0, vocab - 1, vocab // 2], device=DEV), top=32)
            assert torch.equal(r.top_ids, torch.arange(32, device=DEV).expand(3, 32))
            assert r.rank.tolist() == [1, vocab, vocab // 2 + 1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab", [(2, 100_003), (2, 8192), (310, 20_000), (305, 517)])
@pytest.mark.parametrize("kind", ["falling", "rising", "few", "none but one", "steps", "block of equals", "blocks"])
def test_best_scores_however_they_lie(dtype, n, vocab, kind):
    """The largest scores next to each other, far fewer scores than asked for, more equal ones than a list holds: in rows of one CTA
    and of several."""
    ids = torch.arange(vocab, device=DEV).double()
    if kind == "falling":
        x = -ids / 64
    elif kind == "rising":
        x = ids / 64
    elif kind == "few":
        x = torch.where(ids % (vocab // 5) == 3, ids / vocab, -math.inf)
    elif kind == "none but one":
        x = torch.where(ids == vocab - 2, 1.0, -math.inf)
    elif kind == "steps":
        x = (ids * 7919 % vocab * 8 / vocab).floor()
    elif kind == "block of equals":
        x = torch.where((ids > vocab / 3) & (ids < vocab / 2), 2.0, 1.0)
        x[vocab // 2 + 5] = 3.0
    else:
        x = torch.where(ids < vocab // 2, (ids / 700).floor() % 3, 0.0) + (ids % 700 == 0)
    x = x.to(dtype).expand(n, vocab).contiguous()
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen(1))
    for top in (1, 7, 32):
        r = T.token_logprobs(x, targets, top=top)
        want = torch.sort(x[:1].float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids, want.expand(n, top)), (kind, top)
    assert torch.equal(r.rank, _want(x, targets, 1.0, 1)[3])


def test_logprobs_with_nan_infinity_and_bad_targets():
    x = torch.randn(6, 3000, device=DEV, generator=gen(2))
    x[0, 5], x[1, 7], x[2, 2999] = math.nan, math.inf, math.nan
    targets = torch.tensor([1, 2, 3, 3000, -7, -100], device=DEV)
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    r = T.token_logprobs(x, targets, top=4, errors=errors)
    assert r.logprob[:5].isnan().all() and r.lse[:3].isnan().all() and r.entropy[:3].isnan().all()
    assert r.lse[3:5].isfinite().all() and r.rank[3:].tolist() == [0, 0, 0] and errors.item() == 1
    order = torch.sort(torch.where(x.isnan(), -math.inf, x), dim=1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(r.top_ids[:5], order[:5]) and (r.top_ids[5] == -1).all() and r.logprob[5] == 0


def _want_grad(x, targets, scale, lse, ent, g, h):
    keep = (targets >= 0) & (targets < x.shape[1])
    lse, ent = lse.double(), ent.double()
    scale = f32(scale)
    logp = x.double() * scale - lse[:, None]
    p = logp.exp()
    w = -p
    w[torch.arange(len(x)), targets.clamp(0, x.shape[1] - 1)] += 1.0
    size = p.clone()
    size[torch.arange(len(x)), targets.clamp(0, x.shape[1] - 1)] += 1.0
    plogp = torch.special.entr(p)
    out = g.double()[:, None] * w + h.double()[:, None] * (plogp - p * ent[:, None])
    size = g.double().abs()[:, None] * size + h.double().abs()[:, None] * (plogp.abs() + p * ent.abs()[:, None])
    dead = ~keep | (lse == -math.inf)
    out[dead] = 0.0
    size[dead] = 0.0
    return out * scale, size * scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["plain", "masked", "sharp"])
@pytest.mark.parametrize("n,vocab,pad,out", [(1, 1, 0, None), (5, 31, 0, None), (6, 1000, 24, None), (9, 1025, 0, "other"), (8, 14_951, 57, None), (7, 14_951, 0, "self"),
                                             (3, 70_001, 3, "other"), (200, 4096, 0, "self")])
def test_logprobs_grad(dtype, kind, n, vocab, pad, out):
    x = _scores(n, vocab, dtype, n + vocab, kind, pad)
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen(vocab))
    if n > 5:
        targets[5] = -100
    if n > 7:
        targets[7] = vocab
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    f = T.token_logprobs(x, targets, scale=1.3)
    g, h = torch.randn(n, device=DEV, generator=gen(3)), torch.randn(n, device=DEV, generator=gen(4))
    want, size = _want_grad(x, targets, 1.3, f.lse, f.entropy, g, h)
    # p is off by at most |log p| * 4 * 2^-24 + 2^-21 relatively: below 2e-5 where log p > -60, and nothing elsewhere
    tol = half_step(dtype) * want.abs() + 2e-5 * size
    floor = torch.finfo(dtype).smallest_normal
    room = {None: None, "self": x.clone(), "other": torch.empty(n, vocab + 5, dtype=dtype, device=DEV)[:, 1:1 + vocab]}[out]
    src = room if out == "self" else x
    got = T.token_logprobs_grad(src, targets, f.lse, f.entropy, g, h, scale=1.3, out=room, errors=errors)
    close(got, want, 1.0, tol, floor)
    assert errors.item() == (1 if n > 7 else 0)
    if out is None:
        want, size = _want_grad(x, targets, 1.3, f.lse, f.entropy, g, torch.zeros_like(h))
        close(T.token_logprobs_grad(x, targets, f.lse, None, g, scale=1.3), want, 1.0, half_step(dtype) * want.abs() + 2e-5 * size, floor)
        want, size = _want_grad(x, targets, 1.3, f.lse, f.entropy, torch.zeros_like(g), h)
        close(T.token_logprobs_grad(x, targets, f.lse, f.entropy, None, h, scale=1.3), want, 1.0, half_step(dtype) * want.abs() + 2e-5 * size, floor)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-math.inf, -1e9, -3e38])
def test_a_mask_that_leaves_nothing_gives_no_gradient(dtype, mask):
    x = torch.randn(3, 2051, device=DEV, generator=gen(4)).to(dtype)
    x[1] = mask
    x[2, 5:] = mask
    targets = torch.tensor([7, 8, 2], device=DEV)
    g, h = torch.ones(3, device=DEV), torch.ones(3, device=DEV)
    r = T.token_logprobs(x, targets)
    got = T.token_logprobs_grad(x, targets, r.lse, r.entropy, g, h)
    assert (got[1] == 0).all() and (got[2, 5:] == 0).all() and got.isfinite().all()
    assert r.logprob[1] == -math.inf if mask == -math.inf else abs(r.logprob[1].item() + math.log(2051)) < 2e-4
    p = torch.softmax(x.double(), 1)
    H = torch.special.entr(p).sum(1, keepdim=True)
    for row in (0, 2):
        want = -p[row] - (-torch.special.entr(p[row]) + p[row] * H[row])
        want[targets[row]] += 1
        assert ((got[row].double() - want).abs() <= half_step(dtype) * want.abs() + 2e-4 * p[row] + 1e-6 * (1 if dtype == torch.float32 else 0)).all()


def _exact_grad(x, targets, scale, g, h):
    """From the scores alone, the differences to the largest one first: the gradient, and the sum of its terms' sizes."""
    z = (x.double() - x.double().amax(1, keepdim=True)) * f32(scale)
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    p = logp.exp()
    hot = torch.zeros_like(p).scatter_(1, targets[:, None], 1.0)
    plogp, H = torch.special.entr(p), torch.special.entr(p).sum(1, keepdim=True)
    want = g.double()[:, None] * (hot - p) + h.double()[:, None] * (plogp - p * H)
    size = g.double().abs()[:, None] * (hot + p) + h.double().abs()[:, None] * (plogp + p * H)
    return want * f32(scale), size * f32(scale), p


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("base,scale", [(-1e30, 1.0), (-1e9, 1.0), (-1e9, 0.7), (-65_000.0, 1.0), (-300.0, 1.3), (3e4, 1.0), (1e6, 1.0), (1e6, 0.7), (1e9, 1.0), (1e30, 1.0),
                                        (-20.0, 1e5), (20.0, 1e5), (-3.0, 1e20)])
@pytest.mark.parametrize("n,vocab,own", [(3, 11, False), (2, 30_000, True), (150, 2051, False)])
def test_logprobs_grad_far_from_zero(dtype, base, scale, n, vocab, own):
    """With the rest of lse the gradient is that of the scores themselves, wherever they lie: p is off by a few roundings of log p, as around
    zero.  Without it, p is off by half a step of lse more, and where lse is beyond 1e6 the row says so."""
    if dtype == torch.float16 and abs(base) > 65_504:
        base = math.copysign(6e4, base)
    x = torch.full((n, vocab), base, device=DEV).to(dtype)
    step = x[0, 0].float().abs().item() * torch.finfo(dtype).eps
    if step * scale < 64:
        x = (x.float() + torch.randint(-3, 4, (n, vocab), device=DEV, generator=gen(9)) * step).to(dtype)
    targets = torch.randint(0, vocab, (n,), device=DEV, generator=gen(3))
    g, h = torch.randn(n, device=DEV, generator=gen(4)) / scale, torch.randn(n, device=DEV, generator=gen(5)) / scale
    want, size, p = _exact_grad(x, targets, scale, g, h)
    r = T.token_logprobs(x, targets, scale=scale)
    assert len(r) == 6 and r.lse_rest.dtype == torch.float32
    lse = r.lse.double()
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    tol, floor = half_step(dtype) * want.abs() + 2e-5 * size, torch.finfo(dtype).smallest_normal
    to = x.clone() if own else None
    close(T.token_logprobs_grad(to if own else x, targets, r.lse, r.entropy, g, h, scale=scale, errors=errors, lse_rest=r.lse_rest, out=to), want, 1.0, tol, floor)
    assert errors.item() == 0
    got = T.token_logprobs_grad(x, targets, r.lse, r.entropy, g, h, scale=scale, errors=errors)
    if lse.abs().max() <= 1e6:
        close(got, want, 1.0, tol + torch.expm1(2 ** -24 * 2 * lse.abs())[:, None] * size * 20, floor)   # (p log p: its own slope, below 20, more)
        assert errors.item() == 0
    else:
        assert (got == 0).all() if lse.max() < 0 else got.isnan().all()
        assert errors.item() == 4
        with pytest.raises(ValueError, match="lse_rest"):
            T.check_errors(errors)


def test_rows_with_an_infinite_lse_have_no_gradient_to_give():
    """-inf: nothing is left, zeros.  +inf, where scale times the scores leaves float32: NaN, and it is reported."""
    x = torch.full((3, 100), -math.inf, device=DEV)
    x[1] = 3e38
    x[2] = torch.randn(100, device=DEV, generator=gen(1))
    targets, g = torch.tensor([1, 2, 3], device=DEV), torch.ones(3, device=DEV)
    r = T.token_logprobs(x, targets, scale=2.0)
    for rest in (None, r.lse_rest):
        errors = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = T.token_logprobs_grad(x, targets, r.lse, None, g, scale=2.0, errors=errors, lse_rest=rest)
        assert (got[0] == 0).all() and got[1].isnan().all() and errors.item() == 4
        want, size, _ = _exact_grad(x[2:], targets[2:], 2.0, g[2:], 0 * g[2:])
        close(got[2:], want, 1.0, 2e-5 * size)


@pytest.mark.parametrize("n,kind", [(7, "one"), (600, "half"), (1536, "one"), (1537, "half"), (70_000, "half")])
def test_ids_of_padding_that_are_most_of_the_list(n, kind):
    """One id far more often than the others: the list is summed in parts, in the same order every time."""
    ids = torch.randint(0, 5000, (n,), device=DEV, generator=gen(n))
    ids[torch.rand(n, device=DEV, generator=gen(1)) < (2.0 if kind == "one" else 0.5)] = 17
    grad = torch.randn(n, 1026, device=DEV, generator=gen(2))
    want, size = _grad_want(grad, ids, 5000, 1.0)
    got = T.embedding_lookup_grad(grad, ids, 5000)
    close(got, want, 1.0, 2 ** -24 * want.abs() + (n + 4) * 2 ** -24 * size, floor=1e-37)
    assert torch.equal(got, T.embedding_lookup_grad(grad, ids, 5000))


def test_logprobs_gradient_is_the_slope():
    """Central differences of the 64-bit definition with step e: off by e^2 / 6 of a third derivative below 2, and by what fp32 makes
    of the gradient itself."""
    x = torch.randn(4, 50, device=DEV, generator=gen(1))
    targets = torch.tensor([3, 0, 49, 20], device=DEV)
    g, h = torch.randn(4, device=DEV, generator=gen(3)), torch.randn(4, device=DEV, generator=gen(4))
    f = T.token_logprobs(x, targets)
    got = T.token_logprobs_grad(x, targets, f.lse, f.entropy, g, h).double()

    def value(v):
        logp = torch.log_softmax(v, 1)
        return (g.double() * logp.gather(1, targets[:, None])[:, 0] + h.double() * torch.special.entr(logp.exp()).sum(1)).sum()
    for seed in range(5):
        d = torch.randn(4, 50, device=DEV, generator=gen(10 + seed)).double()
        e = 1e-4
        slope = (value(x.double() + e * d) - value(x.double() - e * d)) / (2 * e)
        assert abs((got * d).sum() - slope).item() < 200 * 2e-5


# ------------------------------------------------------------------------------------- streams, graphs, large offsets
def test_on_a_side_stream_and_in_a_graph():
    g = gen(9)
    table = torch.randn(1000, 64, device=DEV, generator=g)
    ids = torch.randint(0, 1000, (300,), device=DEV, generator=g)
    targets = torch.randint(0, 1000, (300,), device=DEV, generator=g)

    def chain():
        rows = T.embedding_lookup(table, ids, scale=2.0)
        logits = rows @ table.t()
        f = T.token_logprobs(logits, targets, top=3)
        dx = T.token_logprobs_grad(logits, targets, f.lse, f.entropy, torch.ones_like(f.lse), f.entropy)
        return f.logprob, f.top_ids, T.embedding_lookup_grad(dx @ table, ids, 1000, scale=2.0)
    want = [t.clone() for t in chain()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(chain())
        graphs.append(graph)
    targets.add_(1).remainder_(1000)
    want = [t.clone() for t in chain()]
    for graph in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_what_is_written_to_counts_as_modified():
    """What autograd has saved for a backward pass is refused there once a call has written over it."""
    x, ids = torch.randn(4, 8, device=DEV), torch.arange(4, device=DEV)
    w = torch.ones(8, device=DEV, requires_grad=True)
    loss = (x * w).sum()
    r = T.token_logprobs(x, ids)
    T.token_logprobs_grad(x, ids, r.lse, None, torch.ones(4, device=DEV), out=x)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()
    for accumulate in (False, True):
        loss = (x * w).sum()
        T.embedding_lookup_grad(torch.ones(4, 8, device=DEV), ids, 4, out=x, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="modified"):
            loss.backward()


def test_offsets_beyond_32_bits():
    rows, dim = 2_200_000, 1024                      # 2.25e9 elements
    table = torch.empty(rows, dim, dtype=torch.bfloat16, device=DEV)
    table[-3:] = torch.randn(3, dim, device=DEV, generator=gen(1)).to(torch.bfloat16)
    ids = torch.tensor([rows - 1, rows - 3, rows - 1], device=DEV)
    assert torch.equal(T.embedding_lookup(table, ids), table[ids])
    grad = torch.randn(3, dim, device=DEV, generator=gen(2)).to(torch.bfloat16)
    out = T.embedding_lookup_grad(grad, ids, rows, out=table)
    assert torch.equal(out[-3], grad[1]) and (out[:-3:100_000] == 0).all() and (out[-2] == 0).all()
    close(out[-1], grad[0].double() + grad[2].double(), 2 ** -8, (grad[0].double() + grad[2].double()).abs(), 2 ** -20)
    logits = table.view(-1)[: 2200 * 1_024_000].view(2200, 1_024_000)
    logits[-1].normal_()
    targets = torch.full((2200,), -100, device=DEV)
    targets[-1] = 77
    r = T.token_logprobs(logits, targets, top=2)
    assert r.top_ids[-1, 0] == logits[-1].float().argmax()
    d = T.token_logprobs_grad(logits, targets, r.lse, None, torch.ones(2200, device=DEV), out=logits)
    assert abs(d[-1].float().sum().item()) < 1024 * 1000 * 2 ** -9 * 1e-3 and (d[-2] == 0).all()


@pytest.mark.parametrize("own", [False, True])
def test_rows_of_scores_beyond_2_to_the_31_elements(own):
    """Every result of the rows that begin, or go on, behind the 2^31st element, against the definition: a target, a score or a result taken from an offset
    cut to 32 bits would be another row's."""
    n, vocab = 2104, 1_024_000                                   # the 2098th row holds element 2^31
    logits = torch.zeros(n, vocab, dtype=torch.bfloat16, device=DEV)
    rows = [0, 2096, 2097, 2098, 2103]
    for k, row in enumerate(rows):
        logits[row] = torch.randn(vocab, device=DEV, generator=gen(row)) + k
    targets = torch.full((n,), -100, device=DEV)
    at = torch.tensor(rows, device=DEV)
    targets[at] = torch.tensor([5, vocab - 1, 700_000, 0, 512_001], device=DEV)
    x = logits[at].clone()
    r = T.token_logprobs(logits, targets, top=3)
    logprob, ent, lse, rank, best, ids = _want(x, targets[at], 1.0, 3)
    close(r.lse[at], lse, 2e-5, 1 + lse.abs())
    close(r.logprob[at], logprob, 2e-5, 1 + lse.abs() + logprob.abs())
    close(r.entropy[at], ent, 2e-5, 1 + ent + math.log(vocab))
    assert torch.equal(r.rank[at], rank) and torch.equal(r.top_ids[at], ids)
    g = torch.randn(n, device=DEV, generator=gen(1))
    want, size = _want_grad(x, targets[at], 1.0, r.lse[at], r.entropy[at], g[at], 0.5 * g[at])
    got = T.token_logprobs_grad(logits, targets, r.lse, r.entropy, g, 0.5 * g, lse_rest=r.lse_rest, out=logits if own else None)
    close(got[at], want, 1.0, half_step(torch.bfloat16) * want.abs() + 2e-5 * size + torch.expm1(2 ** -23 * lse.abs())[:, None] * size, torch.finfo(torch.bfloat16).smallest_normal)
    between = torch.ones(n, dtype=torch.bool, device=DEV)
    between[at] = False
    assert not got[between].any()
