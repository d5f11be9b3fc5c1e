"""GPU: layers of different sizes called by several host threads at once."""
import threading

import pytest
import torch

from mini_qwen_b200.kernels import moe_layer_small, w8a8_moe_layer_small

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer(kind, T, H, I, E, K):
    g = torch.Generator(device=DEV).manual_seed(T + E)
    x = torch.randn(T, H, generator=g, device=DEV).bfloat16()
    router = torch.randn(E, H, generator=g, device=DEV).bfloat16()
    if kind == "dense":
        w13 = (torch.randn(E, 2 * I, H, generator=g, device=DEV) * H ** -0.5).bfloat16()
        w2 = (torch.randn(E, H, I, generator=g, device=DEV) * I ** -0.5).bfloat16()
        return lambda: moe_layer_small(x, router, w13, w2, K)
    w13 = torch.randint(-127, 128, (E, 2 * I, H), generator=g, device=DEV, dtype=torch.int8), torch.full((E, 2 * I), 1e-3, device=DEV)
    w2 = torch.randint(-127, 128, (E, H, I), generator=g, device=DEV, dtype=torch.int8), torch.full((E, H), 1e-3, device=DEV)
    return lambda: w8a8_moe_layer_small(x, router, w13, w2, K)


@pytest.mark.parametrize("kind", ["dense", "w8"])
def test_a_smaller_call_takes_nothing_from_a_larger_one(kind):
    """The kernel of one to eight tokens is the same for every size; its shared memory goes by the tokens and the experts."""
    calls = [layer(kind, 8, 128, 64, 1000, 32), layer(kind, 1, 128, 64, 4, 1), layer(kind, 8, 128, 64, 500, 16),
             layer(kind, 2, 128, 64, 8, 2)]
    refs = [call() for call in calls]
    torch.cuda.synchronize()
    start, failures = threading.Barrier(len(calls)), []

    def hammer(call, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for i in range(400):
                    out = call()
                    if i % 50 == 0 and not torch.equal(out, ref):
                        failures.append("another result")
        except Exception as e:                            # noqa: BLE001 - reported below, from the test's own thread
            failures.append(e)

    threads = [threading.Thread(target=hammer, args=pair) for pair in zip(calls, refs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures, failures[0]
