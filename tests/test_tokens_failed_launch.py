"""The token operators when one of their launches fails: the call returns the error, nothing is launched behind the failed launch, and the next
call is as good as the first.  On the CPU (fake_cuda_util)."""
import sys

import pytest

import fake_cuda_util as F


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return F.build_fake(tmp_path_factory.mktemp("fake"))


CALLS = ["lookup", "lookup_grad_none", "lookup_grad_short", "lookup_grad", "lookup_grad_long", "logprobs", "logprobs_grad", "table", "table_few", "table_fp32", "table_grad",
         "table_grad_fp32", "table_grad_fp16_few"]


@pytest.mark.parametrize("call", CALLS)
def test_a_failed_launch_ends_the_call(fake, call):
    F.run_child(__file__, fake, call)


def _calls(lib, name):
    """A function that makes the call once and returns its status, and how many launches it makes."""
    import numpy as np
    p = F.p
    n, rows, D = 300, 700, 64
    x, ids, f, out, errors = F.dev((rows, D), np.float32), F.dev(70_000, np.int64), F.dev(n, np.float32), F.dev((rows, D), np.float32), F.dev(1, np.int32)
    if name == "lookup":
        return lambda: lib.pbg_embedding_lookup(p(x), D, rows, D, 0, p(ids), n, 1.0, p(out), p(errors), None), 1
    if name.startswith("lookup_grad"):
        m = {"lookup_grad_none": 0, "lookup_grad_short": 1536, "lookup_grad": 1537, "lookup_grad_long": 70_000}[name]
        g, size = F.dev((m + 1, 4), np.float32), lib.pbg_embedding_lookup_grad_workspace(m, rows, 4)
        ws = F.dev(size + 256, np.uint8)
        return lambda: lib.pbg_embedding_lookup_grad(p(g), 4, p(ids), m, rows, 4, 0, 1.0, p(out), 4, 0, p(ws), size, p(errors), None), {0: 1, 1536: 1, 1537: 3, 70_000: 6}[m]
    logits, rank, best = F.dev((n, 100), np.float32), F.dev(n, np.int64), F.dev((n, 8), np.int64)
    if name == "logprobs":
        return lambda: lib.pbg_token_logprobs(p(logits), 100, n, 100, 0, p(ids), -100, 1.0, 8, p(f), p(f), p(f), p(rank), p(best), p(best), p(errors), None), 1
    if name == "logprobs_grad":
        return lambda: lib.pbg_token_logprobs_grad(p(logits), 100, n, 100, 0, p(ids), -100, 1.0, p(f), p(f), p(f), p(f), p(logits), 100, p(errors), None), 1
    dtype = 0 if "fp32" in name or name == "table_few" else 2 if "fp16" in name else 1
    few = 4 if "few" in name else n
    grad = int("grad" in name)
    size = lib.pbg_table_logprobs_workspace(few, rows, D, dtype, grad)
    ws = F.dev(size + 256, np.uint8)
    if not grad:
        count = {"table": 2, "table_few": 2, "table_fp32": 4}[name]
        return lambda: lib.pbg_table_logprobs(p(x), D, few, p(x), D, rows, D, dtype, p(ids), -100, 1.0, p(f), p(f), p(f), p(ws), size, p(errors), None), count
    # the queries' copy (and what it is scaled by), dz, dQ, dW, and the join where dQ is split
    least = {"table_grad": 4, "table_grad_fp32": 5, "table_grad_fp16_few": 5}[name]
    return lambda: lib.pbg_table_logprobs_grad(p(x), D, few, p(x), D, rows, D, dtype, p(ids), -100, 1.0, p(f), p(f), p(f), p(f), p(x), p(out), p(ws), size, p(errors), None), least


def main(fake_so, name):
    fake, L, lib = F.load(fake_so)
    call, launches = _calls(lib, name)
    fake.fake_arm(0, 0)
    assert call() == L.PBG_OK
    many = fake.fake_launches()
    assert many == launches or ("table_grad" in name and many == launches + 1) or (name == "lookup_grad_long" and many >= launches), many
    for at in range(1, many + 1):
        fake.fake_arm(at, 1)
        assert call() == L.PBG_ERR_CUDA, at
        assert fake.fake_behind_failure() == 0, (at, fake.fake_behind_failure())
        fake.fake_arm(0, 0)
        assert call() == L.PBG_OK and fake.fake_launches() == many, at


if __name__ == "__main__":
    main(*sys.argv[1:])
