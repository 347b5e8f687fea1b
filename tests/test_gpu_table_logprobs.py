"""Log probabilities over all rows of a table and their gradients, against the definition in 64 bits.

Tolerances.  u = 2^-24.
  - A score is a dot product of dim exact products (16-bit operands) added up in fp32, at worst truncated: off by dim * 2 u of the sum of
    the products' sizes; float32 operands are two fp16 planes, which drop 2^-22 of a product and round each operand by 2^-22: 3 * 2^-22
    more.  E = (dim * 2^-23 + 3 * 2^-22) * max |q||w| summed bounds a score's error, and with it that of lse and log p (all scores off by E at
    most; softmax moves by no more than its scores), beside 2e-5 of 1 + |lse| for the sums as in the tests of scores in memory; the
    entropy moves by at most 2 E times its own slope, |log p| + H <= 40 where p counts.
  - dz is off by p (E + 2e-5) relatively and rounded by half a step of the operands' type (float32: two planes, 2^-22); the products
    with the table and the queries carry that as a sum of sizes, and 2^-23 per term of fp32 adding."""
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
    return float(torch.tensor(scale, dtype=torch.float32))


def half_step(t):
    return torch.finfo(t).eps / 2


def inputs(n, rows, dim, dtype, seed, spread=1.0):
    g = gen(seed)
    table = (torch.randn(rows, dim, device=DEV, generator=g) / math.sqrt(dim)).to(dtype)
    targets = torch.randint(0, rows, (n,), device=DEV, generator=g)
    queries = (spread * (torch.randn(n, dim, device=DEV, generator=g) + 2 * table[targets].float())).to(dtype)
    return queries, table, targets


def scores(q, t, scale):
    """64-bit scores, and the bound E per row on the error of one."""
    z = q.double() @ t.double().T * f32(scale)
    size = (q.double().abs() @ t.double().abs().T).amax(1) * scale
    dim = q.shape[1]
    return z, size * (dim * 2 ** -23 + (3 * 2 ** -22 if q.dtype == torch.float32 else 0))


def want_forward(z, targets):
    lse = torch.logsumexp(z, 1)
    logp = z - lse[:, None]
    return logp.gather(1, targets[:, None])[:, 0], torch.special.entr(logp.exp()).sum(1), lse


def check_forward(q, t, targets, scale, ignore=()):
    r = T.table_logprobs(q, t, targets, scale=scale)
    keep = torch.ones(len(q), dtype=torch.bool, device=DEV)
    keep[list(ignore)] = False
    z, E = scores(q[keep], t, scale)
    logprob, ent, lse = want_forward(z, targets[keep])
    tol = E + 2e-5 * (1 + lse.abs())
    assert ((r.lse[keep].double() - lse).abs() <= tol).all()
    assert ((r.logprob[keep].double() - logprob).abs() <= 2 * tol + 2e-5 * logprob.abs()).all()
    assert ((r.entropy[keep].double() - ent).abs() <= 80 * E + 2e-5 * (1 + ent + math.log(len(t)))).all()
    for x in r:
        assert (x[~keep] == 0).all() and x.dtype == torch.float32
    return r


SHAPES = [(1, 1, 1), (1, 300, 8), (3, 64, 64), (5, 65, 33), (127, 255, 40), (129, 257, 72), (7, 20_011, 400), (200, 1000, 1), (64, 3000, 520), (300, 5000, 100), (1000, 14_951, 400), (5, 700, 2112), (300, 900, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", SHAPES)
def test_forward(dtype, n, rows, dim):
    q, t, targets = inputs(n, rows, dim, dtype, n + rows)
    ignore = [4] if n > 4 else []
    targets[ignore] = -100
    check_forward(q, t, targets, 0.9, ignore)


def check_grad(q, t, targets, scale, g, h, r, got, dead=()):
    dq, dt = got
    keep = torch.ones(len(q), dtype=torch.bool, device=DEV)
    keep[list(dead)] = False
    qk, tk = q[keep], targets[keep]
    z, E = scores(qk, t, scale)
    logp = z - r.lse[keep].double()[:, None]
    p = logp.exp()
    hot = torch.zeros_like(p)
    hot[torch.arange(len(p), device=DEV), tk] = 1.0
    gk = g[keep].double()[:, None] if g is not None else torch.zeros(len(p), 1, device=DEV, dtype=torch.float64)
    hk = h[keep].double()[:, None] if h is not None else torch.zeros_like(gk)
    H = r.entropy[keep].double()[:, None]
    w = scale * (gk * (hot - p) + hk * (torch.special.entr(p) - p * H))
    size = scale * (gk.abs() * (hot + p) + hk.abs() * (torch.special.entr(p).abs() + p * H))
    err = size * (E[:, None] * 2 + 2e-5) + scale * hk.abs() * p * E[:, None] + w.abs() * (2 ** -22 if q.dtype == torch.float32 else half_step(q.dtype))
    if q.dtype != torch.bfloat16:
        # a power of two brings the bound of dz to 2^14; half a step of the smallest half-precision numbers is 2^-25 of 1
        bound = scale * ((g[keep].abs().max().item() if g is not None else 0) + 23 * (h[keep].abs().max().item() if h is not None else 0))
        err = err + bound * 2 ** -38
    A, Q = t.double(), qk.double()
    planes = 3 * 2 ** -22 if q.dtype == torch.float32 else 0
    floor = torch.finfo(q.dtype).smallest_normal
    want = w @ A
    tol = err @ A.abs() + (w.abs() @ A.abs()) * (len(t) * 2 ** -23 + planes) + want.abs() * half_step(q.dtype) + floor
    assert ((dq[keep].double() - want).abs() <= tol).all(), ((dq[keep].double() - want).abs() - tol).max()
    want = w.T @ Q
    tol = err.T @ Q.abs() + (w.abs().T @ Q.abs()) * (len(qk) * 2 ** -23 + planes) + want.abs() * half_step(q.dtype) + floor
    assert ((dt.double() - want).abs() <= tol).all(), ((dt.double() - want).abs() - tol).max()
    assert (dq[~keep] == 0).all() and dq.dtype == q.dtype and dt.dtype == t.dtype


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", SHAPES)
def test_gradients(dtype, n, rows, dim):
    q, t, targets = inputs(n, rows, dim, dtype, n + rows)
    dead = [x for x in (4, 6) if x < n]
    if n > 4:
        targets[4] = -100
        q[4] = math.nan                                     # what stands in padding does not matter
    if n > 6:
        targets[6] = rows
        q[6] = math.inf
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    r = T.table_logprobs(q, t, targets, scale=1.1)
    g, h = torch.randn(n, device=DEV, generator=gen(1)) / n, torch.randn(n, device=DEV, generator=gen(2)) / n
    g[dead] = math.nan
    check_grad(q, t, targets, 1.1, g, h, r, T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, g, h, scale=1.1, errors=errors), dead)
    assert errors.item() == (1 if n > 6 else 0)
    check_grad(q, t, targets, 1.1, g, None, r, T.table_logprobs_grad(q, t, targets, r.lse, None, g, scale=1.1), dead)
    check_grad(q, t, targets, 1.1, None, h, r, T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, None, h, scale=1.1), dead)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,first", [(80, 0), (80, 8), (77, 0), (80, 1)])
def test_strides(dtype, width, first):
    q, t, targets = inputs(50, 700, width, dtype, width)
    q, t = q[:, first:first + 64], t[:, first:first + 64]
    r = check_forward(q, t, targets, 1.0)
    g = torch.ones(50, device=DEV)
    check_grad(q, t, targets, 1.0, g, None, r, T.table_logprobs_grad(q, t, targets, r.lse, None, g))
    same = q[:1].expand(50, 64)
    r2 = check_forward(same, t, targets, 1.0)
    check_grad(same, t, targets, 1.0, g, None, r2, T.table_logprobs_grad(same, t, targets, r2.lse, None, g))


@pytest.mark.parametrize("dtype", TYPES)
def test_the_last_columns_of_wider_rows(dtype):
    """Rows that end where the memory does, in operands read where they lie."""
    q, t, targets = inputs(200, 700, 80, dtype, 80)
    q, t = q[:, 40:], t[:, 40:]
    r = check_forward(q, t, targets, 1.0)
    g = torch.ones(200, device=DEV)
    check_grad(q, t, targets, 1.0, g, None, r, T.table_logprobs_grad(q, t, targets, r.lse, None, g))


def test_float32_operands_of_any_size():
    """Both planes are scaled by the largest element: tables of tiny and of large numbers come out as accurately."""
    q, t, targets = inputs(40, 900, 96, torch.float32, 5)
    for a, b in ((1e-12, 1e12), (1e15, 1e-15), (3e-20, 1e19), (1.0, 1e-30)):
        r = check_forward(q * a, t * b, targets, 1.0)
        g = torch.ones(40, device=DEV)
        check_grad(q * a, t * b, targets, 1.0, g, None, r, T.table_logprobs_grad(q * a, t * b, targets, r.lse, None, g))
    zero = T.table_logprobs(q * 0, t, targets)
    assert (zero.entropy - math.log(900)).abs().max() < 1e-5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [7, 100, 300])
def test_nan_and_infinity_stay_in_their_query(dtype, n):
    q, t, targets = inputs(n, 1700, 72, dtype, n)
    q[[2, 4, n - 1], [3, 0, 71]] = 0.5
    clean = T.table_logprobs(q, t, targets)
    q[2, 3], q[4, 0], q[n - 1, 71] = math.nan, math.inf, -math.inf
    bad = torch.zeros(n, dtype=torch.bool, device=DEV)
    bad[[2, 4, n - 1]] = True
    for a, b in zip(T.table_logprobs(q, t, targets), clean):
        assert a[bad].isnan().all() and torch.equal(a[~bad], b[~bad])


@pytest.mark.parametrize("scale,a,b", [(1e-20, 1.0, 1.0), (1e-20, 1e10, 1e10), (1e20, 1e-20, 1.0), (1.0, 1e-36, 1e36), (1.0, 1e36, 1e-36), (1e20, 1e-35, 1e15)])
@pytest.mark.parametrize("n", [7, 300])
def test_scales_and_float32_operands_at_the_ends_of_their_range(n, scale, a, b):
    q, t, targets = inputs(n, 500, 64, torch.float32, n + 1)
    q, t = q * a, t * b
    r = check_forward(q, t, targets, scale)
    g = torch.ones(n, device=DEV)
    check_grad(q, t, targets, f32(scale), g, None, r, T.table_logprobs_grad(q, t, targets, r.lse, None, g, scale=scale))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_gradients_do_not_vanish(dtype):
    """Most of dz = 2e-5 p lies below the smallest half-precision number, the scaled dz does not."""
    q, t, targets = inputs(100, 500, 64, dtype, 3)
    r = T.table_logprobs(q, t, targets)
    g = torch.full((100,), 2e-5, device=DEV)
    check_grad(q, t, targets, 1.0, g, None, r, T.table_logprobs_grad(q, t, targets, r.lse, None, g))


def test_gradients_are_the_slope():
    """Central differences of the 64-bit definition."""
    q, t, targets = inputs(6, 40, 12, torch.float32, 9)
    r = T.table_logprobs(q, t, targets, scale=1.5)
    g, h = torch.randn(6, device=DEV, generator=gen(1)), torch.randn(6, device=DEV, generator=gen(2))
    dq, dt = T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, g, h, scale=1.5)

    def value(a, b):
        logp = torch.log_softmax(a @ b.T * 1.5, 1)
        return (g.double() * logp.gather(1, targets[:, None])[:, 0] + h.double() * torch.special.entr(logp.exp()).sum(1)).sum()
    e = 1e-4
    for seed in range(4):
        a, b = torch.randn(6, 12, device=DEV, generator=gen(20 + seed)).double(), torch.randn(40, 12, device=DEV, generator=gen(30 + seed)).double()
        Q, W = q.double(), t.double()
        slope = (value(Q + e * a, W + e * b) - value(Q - e * a, W - e * b)) / (2 * e)
        assert abs((dq.double() * a).sum() + (dt.double() * b).sum() - slope).item() < 1e-3


def test_same_bits_and_graphs():
    q, t, targets = inputs(500, 3000, 200, torch.bfloat16, 4)
    g = torch.randn(500, device=DEV, generator=gen(1))

    def step():
        r = T.table_logprobs(q, t, targets)
        return (*r, *T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, g, r.lse))
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    targets.copy_(targets.roll(1))
    q.mul_(0.5)
    want = step()
    for graph in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_and_nothing_to_do():
    q, t, targets = inputs(4, 10, 8, torch.float32, 4)
    f = torch.zeros(4, device=DEV)
    for bad in (lambda: T.table_logprobs(q, t[:, :7], targets), lambda: T.table_logprobs(q, t[:0], targets), lambda: T.table_logprobs(q, t, targets[:3]),
                lambda: T.table_logprobs(q, t, targets, scale=0.0), lambda: T.table_logprobs(q, t.t().contiguous().t(), targets),
                lambda: T.table_logprobs_grad(q, t, targets, f, None, None), lambda: T.table_logprobs_grad(q, t, targets, f, None, None, f)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        T.table_logprobs(q, t.half(), targets)
    r = T.table_logprobs(q[:0], t, targets[:0])
    assert r.lse.shape == (0,)
    dq, dt = T.table_logprobs_grad(q[:0], t, targets[:0], f[:0], None, f[:0])
    assert dq.shape == (0, 8) and (dt == 0).all()
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    targets[2] = 10
    r = T.table_logprobs(q, t, targets, errors=errors)
    assert r.logprob[2].isnan() and r.lse.isfinite().all() and errors.item() == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 200])
def test_long_sums_of_one_sign(dtype, dim):
    """2^20 equal terms: what every addition cut off would add up.  dz and the result are rounded by half a step each; parts of 32,768 16-bit
    terms are 2^-13 off at most, 2^14 parts of float32 terms added in float32 2^-11 (half a step each), 32 parts 2^-20."""
    n = (1 << 20) + 3
    g = torch.full((n,), 2.0 ** -8, device=DEV)
    q, t, targets = torch.ones(n, dim, device=DEV, dtype=dtype), torch.zeros(3, dim, device=DEV, dtype=dtype), torch.zeros(n, dtype=torch.long, device=DEV)
    r = T.table_logprobs(q, t, targets)
    assert (r.lse - math.log(3)).abs().max() < 1e-6
    dt = T.table_logprobs_grad(q, t, targets, r.lse, None, g)[1].double()
    want = torch.tensor([2 / 3, -1 / 3, -1 / 3], dtype=torch.float64, device=DEV)[:, None] * n * 2.0 ** -8
    assert ((dt / want - 1).abs() <= (2 * half_step(dtype) + 2 ** -13 + 2 ** -20 if dtype != torch.float32 else 2 ** -11)).all()
    # the same over the table's rows: all of them alike but the target
    t = torch.ones(n, dim, device=DEV, dtype=dtype)
    t[0] = 0
    q, targets, g = torch.zeros(140, dim, device=DEV, dtype=dtype), torch.zeros(140, dtype=torch.long, device=DEV), torch.ones(140, device=DEV)
    r = T.table_logprobs(q, t, targets)
    dq = T.table_logprobs_grad(q, t, targets, r.lse, None, g)[0].double()
    # (p = 1 / n out of an exponential of the rounded lse, off by 2^-23 * 14 and two more roundings; scaled dz have all of their bits)
    err = 2 * half_step(dtype) + 2 ** -13 + 2 ** -20 if dtype != torch.float32 else 2 ** -11
    if dtype == torch.float16:
        err += 2 ** -38 * n                                 # one scale for all of dz: half a step of the smallest numbers, 2^-25 of 2^-13
    assert ((dq / (-(n - 1) / n) - 1).abs() <= err + 16 * 2 ** -23).all()


@pytest.mark.parametrize("dtype,n,rows", [(torch.bfloat16, 70_001, 16_500), (torch.float32, 30_000, 18_100)])
def test_more_queries_than_the_workspace_holds_at_once(dtype, n, rows):
    """The gradient of the scores is kept for pieces of the table, the parts of dQ added up from piece to piece; a sample of the rows of
    both gradients is checked, and the sums over all of them."""
    q, t, targets = inputs(n, rows, 16, dtype, 7)
    r = T.table_logprobs(q, t, targets)
    g = torch.randn(n, device=DEV, generator=gen(1))
    dq, dt = T.table_logprobs_grad(q, t, targets, r.lse, None, g)
    some = torch.arange(0, n, 997, device=DEV)
    z, E = scores(q[some], t, 1.0)
    w = -g[some].double()[:, None] * (z - r.lse[some].double()[:, None]).exp()
    w[torch.arange(len(some), device=DEV), targets[some]] += g[some].double()
    step = half_step(dtype) if dtype != torch.float32 else 2 ** -22
    size = (w.abs() + 2 * g[some].double().abs()[:, None] * (z - r.lse[some].double()[:, None]).exp()) @ t.double().abs()
    tol = size * (step + 2 * E.max() + 2e-5 + rows * 2 ** -23) + (w @ t.double()).abs() * half_step(dtype)
    assert ((dq[some].double() - w @ t.double()).abs() <= tol).all()
    # <dt, x> for a vector x is sum_n <dz_n, t x^T ...>: the table's gradient summed over its rows is sum_n (sum_v dz_nv) q_n, and sum_v dz_nv = 0
    total, each = dt.double().sum(0), (g.double().abs()[:, None] * q.double().abs()).sum(0)
    assert (total.abs() <= 2 * each * (step + half_step(dtype) + 2e-5)).all()
    pick = torch.arange(0, rows, 501, device=DEV)
    want, size = torch.zeros(len(pick), 16, dtype=torch.float64, device=DEV), torch.zeros(len(pick), 16, dtype=torch.float64, device=DEV)
    for part in torch.arange(n, device=DEV).split(4096):
        zz = q[part].double() @ t[pick].double().T
        p = (zz - r.lse[part].double()[:, None]).exp()
        hot = (targets[part][:, None] == pick[None, :]).double()
        want += (g[part].double()[:, None] * (hot - p)).T @ q[part].double()
        size += (g[part].double().abs()[:, None] * (hot + p)).T @ q[part].double().abs()
    assert ((dt[pick].double() - want).abs() <= size * (step + 2 * E.max() + 2e-5 + n * 2 ** -23) + want.abs() * half_step(dtype)).all()


def test_more_partial_sums_than_the_workspace_holds_at_once():
    """The forward pass in pieces of the queries."""
    n, rows = 150_000, 70_000
    q, t, targets = inputs(n, rows, 8, torch.float16, 3)
    r = T.table_logprobs(q, t, targets)
    some = torch.cat((torch.arange(0, n, 2999, device=DEV), torch.tensor([n - 1], device=DEV)))
    z, E = scores(q[some], t, 1.0)
    logprob, ent, lse = want_forward(z, targets[some])
    assert ((r.lse[some].double() - lse).abs() <= E + 2e-5 * (1 + lse.abs())).all()
    assert ((r.logprob[some].double() - logprob).abs() <= 2 * (E + 2e-5 * (1 + lse.abs())) + 2e-5 * logprob.abs()).all()
    assert ((r.entropy[some].double() - ent).abs() <= 80 * E + 2e-5 * (1 + ent + math.log(rows))).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_with_both_ends_of_a_table(dtype):
    """Rows by id, a map, log probabilities over the same table, and the gradient of a policy loss with entropy back to the table and the map;
    against autograd in 64 bits.  Every operator rounds to its type; the bound counts the four roundings on the way to a gradient,
    each relative to the sums of sizes, which the 64-bit graph over absolute values gives."""
    g = gen(11)
    rows, dim, n = 3001, 72, 260
    table = (torch.randn(rows, dim, device=DEV, generator=g) / 8).to(dtype)
    mix = (torch.randn(dim, dim, device=DEV, generator=g) / 8).to(dtype)
    ids, targets = torch.randint(0, 40, (n,), device=DEV, generator=g), torch.randint(0, rows, (n,), device=DEV, generator=g)
    targets[::17] = -100
    weight = torch.randn(n, device=DEV, generator=g)
    scale = math.sqrt(dim)
    # the step as a program makes it
    x = T.embedding_lookup(table, ids, scale=scale)
    h = x @ mix
    f = T.table_logprobs(h, table, targets)
    gain = torch.full((n,), 0.1, device=DEV)
    dh, dtable = T.table_logprobs_grad(h, table, targets, f.lse, f.entropy, weight, gain)
    dmix, dx = x.t() @ dh, dh @ mix.t()
    T.embedding_lookup_grad(dx, ids, rows, scale=scale, out=dtable, accumulate=True)
    # the same in 64 bits
    W, M = table.double().requires_grad_(), mix.double().requires_grad_()
    keep = targets >= 0
    H = (W[ids] * f32(scale)) @ M
    logp = torch.log_softmax(H @ W.T, 1)[keep]
    loss = (weight[keep].double() * logp.gather(1, targets[keep][:, None])[:, 0]).sum() + 0.1 * torch.special.entr(logp.exp()).sum()
    gW, gM = torch.autograd.grad(loss, (W, M))
    for got, want in ((dtable, gW), (dmix, gM)):
        rel = ((got.double() - want).norm() / want.norm()).item()
        # scores of size s move p by s times the rounding of h: |h| |w| summed is below 30 here
        assert rel < (30 + 4) * half_step(dtype) + 2e-5, rel



@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", [(40, 300, 64), (300, 1000, 100), (200, 3000, 2112)])
def test_a_wait_that_runs_out_leaves_nan(dtype, n, rows, dim):
    """With a limit of 0 every wait of the kernels runs out at once: nothing is loaded or multiplied.  Then no result is left as the memory was, with
    or without an error word, and the next call is as good as the one before."""
    q, t, targets = inputs(n, rows, dim, dtype, 3)
    g = torch.ones(n, device=DEV)
    want = T.table_logprobs(q, t, targets)
    want_grad = T.table_logprobs_grad(q, t, targets, want.lse, want.entropy, g, g)
    errors = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = T.tokens._lib.lib().pbg_table_logprobs_wait_limit(0)
    try:
        for word in (None, errors):
            r = T.table_logprobs(q, t, targets, errors=word)
            assert all(x.isnan().all() for x in r)
            dq, dt = T.table_logprobs_grad(q, t, targets, want.lse, want.entropy, g, g, errors=word)
            assert dq.isnan().all() and dt.isnan().all()
        assert errors.item() == 2
        with pytest.raises(T.tokens._lib.PbgError):
            T.check_errors(errors)
    finally:
        T.tokens._lib.lib().pbg_table_logprobs_wait_limit(before)
    r = T.table_logprobs(q, t, targets, errors=errors)
    assert all(torch.equal(a, b) for a, b in zip(r, want))
    assert all(torch.equal(a, b) for a, b in zip(T.table_logprobs_grad(q, t, targets, want.lse, want.entropy, g, g, errors=errors), want_grad)) and errors.item() == 0


def uneven(n, dim, big, rows=2000):
    """Inputs among which one query and one row of the table are far larger than the rest (the row where no query looks), one of each far smaller; the
    bound E on the others' scores is that of the others."""
    q, t, targets = inputs(n, rows, dim, torch.float32, n + dim)
    q[:, 0] = q[:, 0].abs() + 0.1
    t[7] = 0
    t[7, 0] = -big
    t[11] /= big
    targets[(targets == 7) | (targets == 11)] = 12
    q[5] /= big
    z, E = scores(q, torch.cat((t[:7], t[8:])), 1.0)
    q[3] *= big
    keep = torch.arange(n, device=DEV) != 3
    return q, t, targets, keep, torch.cat((z[:, :7], -big * q[:, :1].double(), z[:, 7:]), 1)[keep], E[keep]


@pytest.mark.parametrize("big", [1e4, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("n,dim", [(16, 72), (17, 72), (17, 400), (140, 33), (1000, 400), (20, 2501), (20, 2052), (20, 9004)])
def test_a_large_row_takes_nothing_from_the_others(n, dim, big):
    """Forward, fp32: what a query gets depends neither on another query's size nor on that of a row it has no score for."""
    q, t, targets, keep, z, E = uneven(n, dim, big)
    r = T.table_logprobs(q, t, targets)
    logprob, ent, lse = want_forward(z, targets[keep])
    tol = E + 2e-5 * (1 + lse.abs())
    assert ((r.lse[keep].double() - lse).abs() <= tol).all()
    assert ((r.logprob[keep].double() - logprob).abs() <= 2 * tol + 2e-5 * logprob.abs()).all()
    assert ((r.entropy[keep].double() - ent).abs() <= 80 * E + 2e-5 * (1 + ent + math.log(len(t)))).all()


def test_float32_queries_in_pieces():
    """More partial sums than the workspace holds at once: every piece takes its own rows' powers of two."""
    n, rows = 150_000, 70_000
    q, t, targets = inputs(n, rows, 8, torch.float32, 3)
    q *= torch.exp(torch.arange(n, device=DEV) % 9 - 4.0)[:, None]
    r = T.table_logprobs(q, t, targets, scale=0.5)
    some = torch.cat((torch.arange(0, n, 2999, device=DEV), torch.tensor([n - 1], device=DEV)))
    z, E = scores(q[some], t, 0.5)
    logprob, ent, lse = want_forward(z, targets[some])
    assert ((r.lse[some].double() - lse).abs() <= E + 2e-5 * (1 + lse.abs())).all()
    assert ((r.logprob[some].double() - logprob).abs() <= 2 * (E + 2e-5 * (1 + lse.abs())) + 2e-5 * logprob.abs()).all()
    assert ((r.entropy[some].double() - ent).abs() <= 80 * E + 2e-5 * (1 + ent + math.log(rows))).all()


@pytest.mark.parametrize("big", [1e4, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("n,dim", [(7, 72), (17, 400), (140, 33), (1000, 400)])
def test_gradients_of_uneven_inputs(n, dim, big):
    """fp32: a query of 1e30 whose gradients are zero, a row of the table where no query looks, a query with gradients of 1e-12 and a row of which every
    query is far.  Each result against the sum of its own terms' sizes: neither what others hold nor a common bound of all dz takes bits from it."""
    q, t, targets, _, _, _ = uneven(n, dim, big)
    t[13] = 0
    t[13, 0] = -400.0
    targets[targets == 13] = 12
    g, h = torch.randn(n, device=DEV, generator=gen(1)) / n, torch.randn(n, device=DEV, generator=gen(2)) / n
    g[3], h[3], g[6], h[6] = 0, 0, 1e-12, 1e-12
    r = T.table_logprobs(q, t, targets)
    dq, dt = T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, g, h)
    keep = torch.arange(n, device=DEV) != 3
    Q, A = q[keep].double(), t.double()
    z = Q @ A.T
    p = (z - r.lse[keep].double()[:, None]).exp()
    hot = torch.zeros_like(p).scatter_(1, targets[keep][:, None], 1.0)
    gk, hk, H = g[keep].double()[:, None], h[keep].double()[:, None], r.entropy[keep].double()[:, None]
    plogp = torch.special.entr(p)
    w = gk * (hot - p) + hk * (plogp - p * H)
    size = gk.abs() * (hot + p) + hk.abs() * (plogp + p * H)
    # each score is off by its own terms' sizes times E's factor, and lse by what that is in the mean under p
    own = (Q.abs() @ A.abs().T) * (dim * 2 ** -23 + 3 * 2 ** -22)
    score = own + (p * own).sum(1, keepdim=True)
    err = size * (2 * score + 2e-5) + hk.abs() * p * score + w.abs() * 2 ** -22
    planes = 3 * 2 ** -22
    # an operand's largest element is brought to 2^39 or above and cut into bf16 planes, whose smallest step is 2^-133: an element is off by at
    # most half a step, 2^-173 of the largest, beside the 2^-24 of its own size (1e-30 among 1e30 is lost)
    least_q, least_t = (x.abs().max().item() * 2.0 ** -173 for x in (q, t))
    want = w @ A
    tol = err @ A.abs() + (w.abs() @ A.abs()) * (len(t) * 2 ** -23 + planes) + want.abs() * 2 ** -24 + 1e-37 + w.abs().sum(1, keepdim=True) * least_t
    assert ((dq[keep].double() - want).abs() <= tol).all()
    want = w.T @ Q
    assert want[13].abs().max() > 1e-37
    tol = err.T @ Q.abs() + (w.abs().T @ Q.abs()) * (n * 2 ** -23 + planes) + want.abs() * 2 ** -24 + 1e-37 + w.abs().sum(0)[:, None] * least_q
    assert ((dt.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", [(5, 3000, 400), (16, 500, 2048), (100, 3000, 72), (300, 5000, 400), (700, 900, 2048), (260, 700, 4096)])
def test_no_log_probability_above_zero(dtype, n, rows, dim):
    """Queries that are sure of their target, whose score is large: log p is between 0 and what the others' scores allow, never on the other
    side."""
    g = gen(n + dim)
    table = (torch.rand(rows, dim, device=DEV, generator=g) / math.sqrt(dim)).to(dtype)
    targets = torch.randint(0, rows, (n,), device=DEV, generator=g)
    for size in (30.0, 300.0, 3000.0):
        q = (size * table[targets].float()).to(dtype)
        r = T.table_logprobs(q, table, targets)
        assert (r.logprob <= 0).all() and (r.entropy >= 0).all()
        z, E = scores(q, table, 1.0)
        logprob, _, lse = want_forward(z, targets)
        assert ((r.logprob.double() - logprob).abs() <= 2 * E + 2e-5 * (1 + lse.abs() + logprob.abs())).all()


@pytest.mark.parametrize("dtype,n", [(torch.float32, 3), (torch.float32, 40), (torch.bfloat16, 3), (torch.float16, 300)])
def test_queries_whose_scores_are_all_minus_infinity(dtype, n):
    """As a row of scores in memory: nothing is left, log probabilities of -inf and no entropy.  (Among float32 queries that are cut into planes an infinity
    has no second part, infinity times 0: NaN.)"""
    q, t, targets = inputs(n, 300, 8, dtype, 4)
    t[:, 0] = 1.0
    q[1, 0] = -math.inf
    r, s = T.table_logprobs(q, t, targets), T.token_logprobs(q.float() @ t.float().T, targets)
    others = torch.arange(n, device=DEV) != 1
    assert r.lse[others].isfinite().all() and r.entropy[others].isfinite().all()
    if dtype == torch.float32 and n > 16:
        assert r.logprob[1].isnan() and r.lse[1].isnan() and r.entropy[1].isnan()
    else:
        assert r.logprob[1] == r.lse[1] == s.logprob[1] == s.lse[1] == -math.inf and r.entropy[1] == s.entropy[1] == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [3, 40, 300])
def test_scores_far_beyond_what_float32_tells_apart(dtype, n):
    """Nothing is left of differences between scores of 1e9; what there is is kept: the largest score has its share of p, no result is NaN and no p above
    1."""
    q, t, targets = inputs(n, 700, 64, dtype, 9)
    q, t = (q.float() * 3e4 / q.float().abs().max()).to(dtype), (t.float() * 3e4 / t.float().abs().max()).to(dtype)
    r = T.table_logprobs(q, t, targets)
    z = q.double() @ t.double().T
    assert z.abs().max() > 1e8
    assert ((r.lse.double() - torch.logsumexp(z, 1)).abs() <= 1e-5 * z.abs().amax(1)).all()
    assert (r.entropy >= 0).all() and (r.entropy <= math.log(700) + 1e-4).all() and (r.logprob <= 0).all() and r.logprob.isfinite().all()
    g = torch.ones(n, device=DEV)
    dq, dt = T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, g, g)
    assert not dq.isnan().any() and not dt.isnan().any()


def lse_size(z):
    return torch.logsumexp(z, 1).abs()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(20, 2048), (100, 4096), (100, 16_384), (20, 65_536)])
def test_probabilities_of_long_rows_add_up_to_one(dtype, n, dim):
    """Scores around 50 whose terms have one sign, so that what a sum cuts off adds up.  The last column of the table is 1: the queries' gradient
    there is the sum of dz, g (1 - sum p).  With z and lse cut alike p is off by the roundings of z and lse, 50 * 3 * 2^-24 < 1e-5, by ex2 and by
    the sums, 2e-6; dz is rounded to 16 bits or more (two planes), the target's by 2^-17 of g."""
    g = gen(dim)
    q, t = torch.rand(n, dim, device=DEV, generator=g).to(dtype), torch.rand(300, dim, device=DEV, generator=g).to(dtype)
    t[:, -1] = 1.0
    targets = torch.randint(0, 300, (n,), device=DEV, generator=g)
    scale = 200.0 / dim
    r = T.table_logprobs(q, t, targets, scale=scale)
    z, _ = scores(q, t, scale)
    # the sums against 64 bits.  An instruction adds 16 products, each cut off at the sum's last bit as the sum itself is: 17 times 2^-25 of the sum so
    # far, half of a part's in the mean, 32 times to a part; the parts are added in fp32 (2^-25 each, in the mean) and lse and z rounded
    tol = lse_size(z) * (32 * 17 * 2 ** -26 + dim / 512 * 2 ** -25 + 4 * 2 ** -24) + 2e-6
    assert ((r.lse.double() - torch.logsumexp(z, 1)).abs() <= tol).all()
    dq, _ = T.table_logprobs_grad(q, t, targets, r.lse, None, torch.full((n,), 1.0 / scale, device=DEV), scale=scale)
    assert dq[:, -1].abs().max() <= 1.2e-5 + 2 ** -17 + 2 ** -17 * 0.5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,rows,dim", [(129, 700, 72), (300, 3000, 400), (40_000, 300, 16)])
def test_gradients_are_as_good_as_their_rounding(dtype, n, rows, dim):
    """A table whose rows have much in common: what rounding takes from dz does not cancel where dz does.  dz keeps two planes, 2^-17 of
    it (fp16: 2^-22 and 2^-39 of its bound), and the results are off by half a step of their own, 1.2e-3 in the mean over the numbers between two
    powers of two (bf16), what a rounding of exact results leaves, and hardly more; with rounded=True by up to three times as much."""
    g = gen(n)
    t = ((1 + torch.randn(rows, dim, device=DEV, generator=g)) / math.sqrt(dim)).to(dtype)
    targets = torch.randint(0, rows, (n,), device=DEV, generator=g)
    q = torch.randn(n, dim, device=DEV, generator=g).to(dtype)
    gr = torch.randn(n, device=DEV, generator=g) / (1 if dtype == torch.float16 else n)
    r = T.table_logprobs(q, t, targets)
    dq, dt = T.table_logprobs_grad(q, t, targets, r.lse, None, gr)
    z = q.double() @ t.double().T
    w = -(z - r.lse.double()[:, None]).exp()
    w[torch.arange(n, device=DEV), targets] += 1
    w *= gr.double()[:, None]
    for got, want in ((dq, w @ t.double()), (dt, w.T @ q.double())):
        rounding = (want.to(dtype).double() - want).norm()
        assert (got.double() - want).norm() <= 1.05 * rounding + 2e-5 * want.norm()
    if dtype == torch.bfloat16:
        d1 = T.table_logprobs_grad(q, t, targets, r.lse, None, gr, rounded=True)[0]
        assert (d1.double() - w @ t.double()).norm() <= 4 * (dq.double() - w @ t.double()).norm()
    one = T.table_logprobs_grad(q[:128], t, targets[:128], r.lse[:128], None, gr[:128])
    two = T.table_logprobs_grad(q[:128], t, targets[:128], r.lse[:128], None, gr[:128], rounded=True)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,rows,dim", [(129, 257, 72), (300, 5000, 100), (1000, 14_951, 400), (40_000, 300, 16)])
def test_rounded_gradients(dtype, n, rows, dim):
    q, t, targets = inputs(n, rows, dim, dtype, n + rows)
    targets[4], q[4] = -100, math.nan
    r = T.table_logprobs(q, t, targets, scale=1.1)
    g, h = torch.randn(n, device=DEV, generator=gen(1)) / n, torch.randn(n, device=DEV, generator=gen(2)) / n
    check_grad(q, t, targets, 1.1, g, h, r, T.table_logprobs_grad(q, t, targets, r.lse, r.entropy, g, h, scale=1.1, rounded=True), [4])
