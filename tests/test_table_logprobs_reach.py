"""What the tensor maps of table_logprobs may reach: the memory of its operands, results and workspace, and no byte behind it.  On the CPU: the
function that encodes a map is replaced by one that notes it."""
import subprocess
import sys

import pytest

import fake_cuda_util as F

SHIM = r"""
typedef unsigned long long u64;
typedef unsigned int u32;
static u64 maps[64][2];
static int count;
extern "C" {
int note_count() { return count; }
u64 note_base(int i) { return maps[i][0]; }
u64 note_bytes(int i) { return maps[i][1]; }
void note_clear() { count = 0; }
// elements of four bytes (type 7) or two; strides of all dimensions but the first, in bytes
static int encode(void *, int type, u32 rank, void *base, const u64 *dims, const u64 *strides, const u32 *, const u32 *, int, int, int, int) {
  u64 bytes = dims[0] * (type == 7 ? 4 : 2);
  for (u32 d = 1; d < rank; ++d) bytes += (dims[d] - 1) * strides[d - 1];
  if (count < 64) { maps[count][0] = (u64)base; maps[count][1] = bytes; ++count; }
  return 0;
}
int cudaGetDriverEntryPoint(const char *, void **p, unsigned long long, int *q) { *p = (void *)encode; if (q) *q = 0; return 0; }
}
"""


@pytest.fixture(scope="module")
def libraries(tmp_path_factory):
    d = tmp_path_factory.mktemp("reach")
    (d / "note.cpp").write_text(SHIM)
    fake = F.build_fake(d)
    subprocess.check_call([F.NVCC, "-shared", "-cudart", "none", "-Xcompiler", "-fPIC", str(d / "note.cpp"), "-o", str(d / "libnote.so")])
    return fake, str(d / "libnote.so")


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("grad", [0, 1])
def test_maps_lie_within_their_buffers(libraries, dtype, grad):
    F.run_child(__file__, *libraries, str(dtype), str(grad))


def main(fake_so, note_so, dtype, grad):
    import ctypes as C

    import numpy as np
    note = C.CDLL(note_so, mode=C.RTLD_GLOBAL)
    note.note_base.restype = note.note_bytes.restype = C.c_ulonglong
    _, L, lib = F.load(fake_so)
    dtype, grad, p = int(dtype), int(grad), F.p
    size = 4 if dtype == 0 else 2
    seen = 0
    # (queries, rows, dim, row stride, first column): rows one behind the other, and columns in the middle and at the end of wider rows
    for n, rows, dim, stride, first in [(40, 300, 64, 64, 0), (40, 300, 40, 80, 40), (300, 700, 40, 80, 0), (300, 700, 8, 72, 64), (300, 700, 72, 144, 72), (300, 700, 100, 100, 0),
                                        (300, 700, 104, 208, 104), (17, 1, 64, 64, 0), (300, 5, 200, 400, 200), (1, 700, 88, 176, 88), (300, 701, 33, 96, 63)]:
        def matrix(r):
            raw = F.dev(r * stride * size, np.uint8)
            return raw.ctypes.data + first * size, raw.ctypes.data, ((r - 1) * stride + first + dim) * size
        q, q0, q_bytes = matrix(n)
        t, t0, t_bytes = matrix(rows)
        ids, f = F.dev(n, np.int64), F.dev(n, np.float32)
        dq, dt = F.dev(n * dim * size, np.uint8), F.dev(rows * dim * size, np.uint8)
        need = lib.pbg_table_logprobs_workspace(n, rows, dim, dtype, grad)
        ws = F.dev(need, np.uint8)
        note.note_clear()
        head = (q, stride, n, t, stride, rows, dim, dtype, p(ids), -100, 1.0)
        tail = (p(ws), need, None, None)
        rc = lib.pbg_table_logprobs_grad(*head, p(f), p(f), p(f), p(f), p(dq), p(dt), *tail) if grad else lib.pbg_table_logprobs(*head, p(f), p(f), p(f), *tail)
        assert rc == L.PBG_OK
        buffers = [(q0, q_bytes), (t0, t_bytes), (ws.ctypes.data, need), (dq.ctypes.data, dq.nbytes), (dt.ctypes.data, dt.nbytes)]
        for i in range(note.note_count()):
            base, nbytes = note.note_base(i), note.note_bytes(i)
            assert any(b <= base and base + nbytes <= b + k for b, k in buffers), (n, rows, dim, stride, first, i, nbytes)
            seen += 1
    assert seen > 0 and note.note_count() < 64


if __name__ == "__main__":
    main(*sys.argv[1:])
