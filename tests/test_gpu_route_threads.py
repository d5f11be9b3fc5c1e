"""GPU: the one-launch routing of batches of different sizes, called by several host threads at once."""
import threading

import pytest
import torch

from mini_qwen_b200 import _cabi
from mini_qwen_b200.kernels.moe_router import moe_route_small, route_small_workspace

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_smaller_batch_takes_nothing_from_a_larger_one():
    """16 tokens of 256 experts take 20 KB of shared memory, one token of 200 takes 4; both run in the same kernel.  The threads
    call the library itself, with tensors that are there before: nothing but the calls takes time."""
    lib, calls, threads, failures = _cabi.load(), [], [], []
    for T, E, K in ((16, 256, 8), (1, 200, 1), (16, 250, 4), (2, 256, 2)):
        g = torch.Generator(device=DEV).manual_seed(E + T)
        x, w = torch.randn(T, 128, generator=g, device=DEV).bfloat16(), torch.randn(E, 128, generator=g, device=DEV).bfloat16()
        ref = moe_route_small(x, w, K, workspace=route_small_workspace(E, x.device))[:5]
        out, ws, stream = [torch.zeros_like(t) for t in ref], route_small_workspace(E, x.device), torch.cuda.Stream()
        ids, weights, perm, inv, off = (t.data_ptr() for t in out)
        args = (x.data_ptr(), 1, w.data_ptr(), 1, None, T, 128, E, K, 0, ws.data_ptr(), ws.numel(), None, ids, weights, perm, inv,
                None, off, None, None, 0, stream.cuda_stream)
        calls.append((args, out, ref, (x, w, ws, stream)))
    torch.cuda.synchronize()
    start = threading.Barrier(len(calls))

    def hammer(args):
        start.wait()
        failures.extend(rc for rc in (lib.mq_route_small(*args) for _ in range(3000)) if rc)

    for args, *_ in calls:
        threads.append(threading.Thread(target=hammer, args=(args,)))
        threads[-1].start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures
    for _, out, ref, _ in calls:
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
