"""What the token operators refuse, on the CPU: tensors on another device than a GPU, wrong types and shapes in the Python
functions, and bad arguments at the C entry points, which return before they touch the device."""
import pytest
import torch

import torchbiggraph_b200 as T
from torchbiggraph_b200 import _lib

BAD, LARGE = _lib.PBG_ERR_BAD_ARGUMENT, _lib.PBG_ERR_TOO_LARGE
P = 4096            # an address that is never read


def test_python_refuses_cpu_tensors():
    x, ids = torch.zeros(3, 4), torch.zeros(3, dtype=torch.long)
    for call in (lambda: T.embedding_lookup(x, ids), lambda: T.embedding_lookup_grad(x, ids, 5), lambda: T.token_logprobs(x, ids),
                 lambda: T.token_logprobs_grad(x, ids, x[:, 0], None, x[:, 0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_python_refuses_forward_mode_tangents():
    """A tangent would be lost without a word: refused, of matrices and of vectors, and only where there is one."""
    from torch.autograd import forward_ad
    x, ids, f = torch.zeros(3, 4), torch.zeros(3, dtype=torch.long), torch.zeros(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: T.embedding_lookup(dual, ids), lambda: T.embedding_lookup_grad(dual, ids, 5), lambda: T.token_logprobs(dual, ids),
                     lambda: T.token_logprobs_grad(dual, ids, f, None, f), lambda: T.table_logprobs(dual, x, ids), lambda: T.table_logprobs_grad(dual, x, ids, f, None, f),
                     lambda: T.tokens._vector("lse", forward_ad.make_dual(f, torch.ones(3)), torch.float32, 3, f.device)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        assert T.tokens._vector("lse", f, torch.float32, 3, f.device) is f
        with pytest.raises(RuntimeError, match="CUDA"):
            T.embedding_lookup(x, ids)


@pytest.mark.parametrize("change,status", [
    (dict(table=None), BAD), (dict(ids=None), BAD), (dict(out=None), BAD), (dict(dim=0), BAD), (dict(dim=65_537), LARGE), (dict(rows=-1), BAD), (dict(rows=0), BAD),
    (dict(rows=2 ** 31), LARGE), (dict(n=-1), BAD), (dict(n=2 ** 31), LARGE), (dict(dtype=3), BAD), (dict(dtype=-1), BAD), (dict(stride=-4), BAD), (dict(scale=float("nan")), BAD)])
def test_lookup_arguments(change, status):
    a = dict(table=P, stride=8, rows=10, dim=8, dtype=0, ids=P, n=4, scale=1.0, out=P)
    a.update(change)
    assert _lib.lib().pbg_embedding_lookup(*a.values(), None, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(grad=None), BAD), (dict(ids=None), BAD), (dict(out=None), BAD), (dict(ws=None), BAD), (dict(ws=P + 16), BAD), (dict(size=10), BAD), (dict(dim=0), BAD),
    (dict(dim=65_537, out_stride=65_537), LARGE), (dict(rows=0), BAD), (dict(n=-1), BAD), (dict(n=2 ** 30 + 1), LARGE), (dict(dtype=5), BAD), (dict(out_stride=7), BAD), (dict(stride=-1), BAD)])
def test_lookup_grad_arguments(change, status):
    L = _lib.lib()
    a = dict(grad=P, stride=8, ids=P, n=4000, rows=10, dim=8, dtype=1, scale=1.0, out=P, out_stride=8, accumulate=0, ws=P, size=L.pbg_embedding_lookup_grad_workspace(4000, 10, 8))
    a.update(change)
    assert L.pbg_embedding_lookup_grad(*a.values(), None, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), BAD), (dict(targets=None), BAD), (dict(lse=None), BAD), (dict(rank=None), BAD), (dict(vocab=0), BAD), (dict(vocab=2 ** 31), LARGE), (dict(n=-1), BAD),
    (dict(n=2 ** 31), LARGE), (dict(dtype=3), BAD), (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("inf")), BAD), (dict(scale=float("nan")), BAD),
    (dict(top=-1), BAD), (dict(top=101), BAD), (dict(top=33), LARGE), (dict(top=2, top_ids=None), BAD), (dict(stride=-1), BAD)])
def test_logprobs_arguments(change, status):
    a = dict(logits=P, stride=100, n=4, vocab=100, dtype=0, targets=P, ignore=-100, scale=1.0, top=0, logprob=P, entropy=P, lse=P, rank=P, top_logprobs=P, top_ids=P)
    a.update(change)
    assert _lib.lib().pbg_token_logprobs(*a.values(), None, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), BAD), (dict(targets=None), BAD), (dict(lse=None), BAD), (dict(entropy=None), BAD), (dict(out=None), BAD), (dict(vocab=0), BAD), (dict(n=-1), BAD),
    (dict(out_stride=99), BAD), (dict(dtype=9), BAD), (dict(scale=0.0), BAD), (dict(vocab=2 ** 31, out_stride=2 ** 31), LARGE), (dict(n=2 ** 31), LARGE)])
def test_logprobs_grad_arguments(change, status):
    a = dict(logits=P, stride=100, n=4, vocab=100, dtype=0, targets=P, ignore=-100, scale=1.0, lse=P, entropy=P, g=P, h=P, out=P, out_stride=100)
    a.update(change)
    assert _lib.lib().pbg_token_logprobs_grad(*a.values(), None, None) == status


def test_nothing_to_do_is_no_error():
    L = _lib.lib()
    assert L.pbg_embedding_lookup(None, 8, 0, 8, 0, None, 0, 1.0, None, None, None) == 0
    assert L.pbg_token_logprobs(None, 8, 0, 8, 0, None, -100, 1.0, 0, *[None] * 8) == 0
    assert L.pbg_token_logprobs_grad(None, 8, 0, 8, 0, None, -100, 1.0, None, None, None, None, None, 8, None, None) == 0
    assert L.pbg_embedding_lookup_grad_workspace(0, 10, 8) == 0


@pytest.mark.gpu
def test_python_refuses_what_does_not_fit():
    x, ids, f = torch.zeros(6, 8, device="cuda"), torch.zeros(6, dtype=torch.long, device="cuda"), torch.zeros(6, device="cuda")
    with pytest.raises(TypeError):
        T.embedding_lookup(x.double(), ids)
    with pytest.raises(TypeError):
        T.embedding_lookup(x, ids.int())
    with pytest.raises(ValueError):
        T.embedding_lookup(x, ids.cpu())
    with pytest.raises(ValueError):
        T.embedding_lookup(x[:0], ids)
    with pytest.raises(ValueError):
        T.embedding_lookup(x.t(), ids)
    with pytest.raises(ValueError):
        T.embedding_lookup(x, ids, scale=float("nan"))
    with pytest.raises(RuntimeError, match="gradient"):
        T.embedding_lookup(x.clone().requires_grad_(), ids)
    with torch.no_grad():
        T.embedding_lookup(x.clone().requires_grad_(), ids)
    with pytest.raises(ValueError):
        T.embedding_lookup_grad(x, ids[:5], 4)
    with pytest.raises(ValueError):
        T.embedding_lookup_grad(x, ids, 0)
    with pytest.raises(ValueError):
        T.embedding_lookup_grad(x, ids, 4, accumulate=True)
    with pytest.raises(ValueError, match="share"):
        T.embedding_lookup_grad(x, ids, 6, out=x)
    with pytest.raises(TypeError):
        T.embedding_lookup_grad(x, ids, 4, out=torch.zeros(4, 8, device="cuda", dtype=torch.half))
    with pytest.raises(ValueError):
        T.embedding_lookup_grad(x, ids, 4, out=torch.zeros(1, 8, device="cuda").expand(4, 8))
    for kw in (dict(top=9), dict(top=-1), dict(scale=0.0), dict(scale=-2.0)):
        with pytest.raises(ValueError):
            T.token_logprobs(x, ids, **kw)
    with pytest.raises(TypeError):
        T.token_logprobs(x, ids, errors=f[:1])
    with pytest.raises(ValueError):
        T.token_logprobs_grad(x, ids, f, None, None)
    with pytest.raises(ValueError):
        T.token_logprobs_grad(x, ids, f, None, f, f)
    with pytest.raises(TypeError):
        T.token_logprobs_grad(x, ids, f.double(), None, f)
    with pytest.raises(ValueError, match="shares"):
        T.token_logprobs_grad(x[:4], ids[:4], f[:4], None, f[:4], out=x[2:])
    assert T.token_logprobs(x[:0], ids[:0], top=3).top_ids.shape == (0, 3)
    assert T.token_logprobs_grad(x[:0], ids[:0], f[:0], None, f[:0]).shape == (0, 8)


TABLE = dict(queries=P, q_stride=8, n=4, table=P, t_stride=8, rows=100, dim=8, dtype=1, targets=P, ignore=-100, scale=1.0)
TABLE_CHANGES = [(dict(queries=None), BAD), (dict(table=None), BAD), (dict(targets=None), BAD), (dict(n=-1), BAD), (dict(rows=0), BAD), (dict(dim=0), BAD), (dict(dim=65_537), LARGE),
                 (dict(n=2 ** 30 + 1), LARGE), (dict(rows=2 ** 31), LARGE), (dict(dtype=7), BAD), (dict(scale=0.0), BAD), (dict(q_stride=-1), BAD), (dict(t_stride=-1), BAD)]


@pytest.mark.parametrize("change,status", TABLE_CHANGES + [(dict(ws=None), BAD), (dict(ws=P + 8), BAD), (dict(size=255), BAD), (dict(lse=None), BAD)])
def test_table_arguments(change, status):
    L = _lib.lib()
    a = dict(TABLE, logprob=P, entropy=P, lse=P, ws=P, size=L.pbg_table_logprobs_workspace(4, 100, 8, 1, 0))
    a.update(change)
    assert L.pbg_table_logprobs(*a.values(), None, None) == status


@pytest.mark.parametrize("change,status", TABLE_CHANGES + [(dict(ws=None), BAD), (dict(ws=P + 8), BAD), (dict(size=255), BAD), (dict(lse=None), BAD), (dict(entropy=None), BAD),
                                                           (dict(dq=None, dt=None), BAD)])
def test_table_grad_arguments(change, status):
    L = _lib.lib()
    a = dict(TABLE, lse=P, entropy=P, g=P, h=P, dq=P, dt=P, ws=P, size=L.pbg_table_logprobs_workspace(4, 100, 8, 1, 1))
    a.update(change)
    assert L.pbg_table_logprobs_grad(*a.values(), None, None) == status


@pytest.mark.parametrize("scale", [1.1e20, 3.4e38, 0.9e-20, 1e-45])
def test_scales_out_of_range(scale):
    """In base 2, or times the powers of two of the operands, such a scale can be infinite or lose its bits."""
    L = _lib.lib()
    a = dict(logits=P, stride=100, n=4, vocab=100, dtype=0, targets=P, ignore=-100, scale=scale)
    assert L.pbg_token_logprobs(*a.values(), 0, P, P, P, P, None, None, None, None) == BAD
    assert L.pbg_token_logprobs_grad(*a.values(), P, P, P, P, P, 100, None, None) == BAD
    a = dict(TABLE, scale=scale)
    assert L.pbg_table_logprobs(*a.values(), P, P, P, P, L.pbg_table_logprobs_workspace(4, 100, 8, 1, 0), None, None) == BAD
    assert L.pbg_table_logprobs_grad(*a.values(), P, P, P, P, P, P, P, L.pbg_table_logprobs_workspace(4, 100, 8, 1, 1), None, None) == BAD
    with pytest.raises(ValueError, match="scale"):
        T.tokens._scale(scale, True)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (7, 131_072, 2048), (16, 65_536, 3000), (17, 65_536, 2048), (1000, 14_951, 400), (5000, 14_951, 400), (4099, 65_536, 2048),
                                        (1 << 20, 131_072, 2048), (1 << 22, 1000, 64), (100, 20_000_000, 64), (30_000, 18_100, 16), (300, 1 << 20, 100), (2000, 500_000, 128)])
def test_workspaces_are_as_large_as_the_header_says(dtype, n, rows, dim):
    L = _lib.lib()
    size, ld, some = (4 if dtype == 0 else 2), (dim + 63) // 64 * 64, 16_384                  # (some: what is rounded up, scales, maxima)
    copies, sums = (n + rows) * ld * size + 4 * (n + rows if dtype == 0 else 0), max(512 << 20, 64 * (rows + 256))
    forward = L.pbg_table_logprobs_workspace(n, rows, dim, dtype, 0)
    if dtype == 0 and n <= 16:
        assert 0 < forward <= 20 * n * 256 + some
    else:
        assert copies <= forward <= copies + sums + 4 * n + some
    planes = 3 if dtype == 0 else 2
    for grad in (1, 2):
        got = L.pbg_table_logprobs_workspace(n, rows, dim, dtype, grad)
        dz = max(2 << 30, 2 * planes * n * 256)
        most = (2.5 if dtype == 0 else 1) * copies + 4 * (n + rows) + dz + max(512 << 20, 4 * n * dim) + some
        assert copies <= got <= most, (got, most)
        if rows * n * planes * 2 <= 1 << 30 and n * dim * 4 <= 1 << 20:                       # small ones do not ask for the limits
            assert got <= (2.5 if dtype == 0 else 1) * copies + 4 * (n + rows) + n * (rows + 64) * planes * 2 + 64 * 4 * n * dim + some


@pytest.mark.parametrize("change,status", [(dict(logits=None), BAD), (dict(lse=None), BAD), (dict(vocab=0), BAD), (dict(top=33), LARGE), (dict(scale=0.0), BAD), (dict(n=2 ** 31), LARGE)])
def test_logprobs_arguments_with_the_rest_of_lse(change, status):
    a = dict(logits=P, stride=100, n=4, vocab=100, dtype=0, targets=P, ignore=-100, scale=1.0, top=0, logprob=P, entropy=P, lse=P, rest=P, rank=P, top_logprobs=P, top_ids=P)
    a.update(change)
    assert _lib.lib().pbg_token_logprobs_wide(*a.values(), None, None) == status


@pytest.mark.parametrize("change,status", [(dict(logits=None), BAD), (dict(lse=None), BAD), (dict(entropy=None), BAD), (dict(out=None), BAD), (dict(out_stride=99), BAD),
                                           (dict(vocab=2 ** 31, out_stride=2 ** 31), LARGE)])
def test_logprobs_grad_arguments_with_the_rest_of_lse(change, status):
    a = dict(logits=P, stride=100, n=4, vocab=100, dtype=0, targets=P, ignore=-100, scale=1.0, lse=P, rest=P, entropy=P, g=P, h=P, out=P, out_stride=100)
    a.update(change)
    assert _lib.lib().pbg_token_logprobs_grad_wide(*a.values(), None, None) == status


@pytest.mark.parametrize("change,status", TABLE_CHANGES + [(dict(ws=None), BAD), (dict(size=255), BAD), (dict(lse=None), BAD), (dict(entropy=None), BAD), (dict(dq=None, dt=None), BAD)])
def test_table_grad_rounded_arguments(change, status):
    L = _lib.lib()
    a = dict(TABLE, n=200, lse=P, entropy=P, g=P, h=P, dq=P, dt=P, ws=P, size=L.pbg_table_logprobs_workspace(200, 100, 8, 1, 2))
    assert a["size"] < L.pbg_table_logprobs_workspace(200, 100, 8, 1, 1)
    a.update(change)
    assert L.pbg_table_logprobs_grad_rounded(*a.values(), None, None) == status


def test_the_limit_of_waits_is_handed_back():
    L = _lib.lib()
    usual = L.pbg_table_logprobs_wait_limit(5)
    assert usual > 1000 and L.pbg_table_logprobs_wait_limit(-1) == 5 and L.pbg_table_logprobs_wait_limit(-1) == usual


@pytest.mark.gpu
def test_python_refuses_a_rest_of_lse_that_does_not_fit():
    x, ids, f = torch.zeros(6, 8, device="cuda"), torch.zeros(6, dtype=torch.long, device="cuda"), torch.zeros(6, device="cuda")
    for bad, error in ((f.double(), TypeError), (f[:5], ValueError), (f.cpu(), ValueError), (f.view(2, 3), ValueError)):
        with pytest.raises(error):
            T.token_logprobs_grad(x, ids, f, None, f, lse_rest=bad)
    # every second element of a vector, as a row that lies apart
    r = T.token_logprobs(x + 3e7, ids)
    apart = torch.stack((r.lse_rest, f), 1)[:, 0]
    assert torch.equal(T.token_logprobs_grad(x + 3e7, ids, r.lse, None, f + 1, lse_rest=apart), T.token_logprobs_grad(x + 3e7, ids, r.lse, None, f + 1, lse_rest=r.lse_rest))
