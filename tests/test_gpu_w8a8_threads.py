"""GPU: W8A8 calls of several host threads at once, and what each of them counts."""
import threading

import pytest
import torch

from mini_qwen_b200 import _cabi
from mini_qwen_b200.kernels import w8a8_gemm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_each_thread_counts_its_own_launches(monkeypatch):
    """One row takes one launch, 100 rows take two, also where both calls have returned before either is counted."""
    w, s = torch.ones(32, 64, dtype=torch.int8, device=DEV), torch.ones(32, device=DEV)
    xs = [torch.ones(rows, 64, device=DEV) for rows in (1, 100)]
    for x in xs:
        w8a8_gemm(x, w, s)
    lib, both, counted = _cabi.load(), threading.Barrier(2), {}
    call = lib.mq_w8a8_linear_x

    def together(*args):
        rc = call(*args)
        both.wait(30)
        return rc

    monkeypatch.setattr(lib, "mq_w8a8_linear_x", together)
    monkeypatch.setattr(_cabi, "count_launches", lambda n: counted.__setitem__(threading.current_thread().name, n))
    threads = [threading.Thread(target=w8a8_gemm, args=(x, w, s), name=str(x.shape[0])) for x in xs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert counted == {"1": 1, "100": 2}
