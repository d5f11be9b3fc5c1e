"""GPU: LinearW8A8 as a module: what it hands to the product."""
import pytest
import torch

import w8a8_reference as R
from mini_qwen_b200.model.layers import LinearW8A8
from mini_qwen_b200.model.layers import linear_w8a8 as module

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [1, 4, 16, 17])
def test_every_call_has_a_status_word(monkeypatch, rows):
    """A small call takes the kernel without waits only where its rows lie on the 16-byte grid; check_status() has to see the
    others too."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    layer = LinearW8A8.from_float(torch.nn.Linear(256, 144, bias=False).to(DEV))
    wide = torch.randn(rows, 300, generator=g, device=DEV).bfloat16()
    words, product = [], module.w8a8_gemm

    def seen(*args, status=None, **kwargs):
        words.append(status)
        return product(*args, status=status, **kwargs)

    monkeypatch.setattr(module, "w8a8_gemm", seen)
    for x in (wide[:, :256].contiguous(), wide[:, 1:257], wide[:, 4:260]):
        q, sx = R.quantize(x)
        R.assert_close(layer(x), R.product(q, sx, layer.qweight, layer.scales))
    assert len(words) == 3 and all(w is layer._status and w is not None for w in words)
    layer.check_status()
    layer._status.fill_(1)                                # what a wait that ran out writes
    with pytest.raises(RuntimeError, match="wait"):
        layer.check_status()
