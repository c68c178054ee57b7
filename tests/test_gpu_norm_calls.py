"""The norm called from several threads, and rows of every length by the form that reads them once.

Tolerances, derived before the first run: half a step of the type (bf16 2^-8, fp16 2^-11, fp32 2^-24) and, for the fp32
statistics, at most 64 additions in a thread and ten joins, 2^-24 each, half of that in the root."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 1e-6
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
STAT = 48 * 2.0 ** -24


def ops():
    from forge import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def test_threads_whose_rows_need_different_shared_memory():
    """One kernel, launched by four threads at once with and without a residual and with rows of different lengths, through
    the C entry point: its argument conversion leaves the threads more time side by side inside the library."""
    from forge import _abi
    lib = _abi.load_library()
    g = gen(1)
    cases = []
    for C in (8192, 6144, 8192, 4096):
        x, r = (torch.randn(1, C, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        w = torch.ones(C, device=DEV, dtype=torch.bfloat16)
        y, h = torch.empty_like(x), torch.empty_like(x)
        res = len(cases) % 2 == 0
        cases.append((x, w, r if res else None, y))
        cases[-1] += ((x.data_ptr(), C, r.data_ptr() if res else None, C, w.data_ptr(), _abi.BF16, _abi.BF16, 1, C, EPS,
                       y.data_ptr(), None, h.data_ptr() if res else None), h)
    bad = []
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()

    def work(i):
        fn, args, st = lib.forge_rmsnorm, cases[i][4], streams[i].cuda_stream
        for _ in range(5000):
            rc = fn(*args, st)
            if rc != 0:
                bad.append((i, rc, lib.forge_last_error()))
                return
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert not bad, bad
    for x, w, r, y, _, h in cases:
        got = ops().rmsnorm(x, w, EPS, residual=r)
        assert torch.equal(got if r is None else got[0], y) and (r is None or torch.equal(got[1], h))
