"""linear's `out` (no GPU): a tensor that is not on the projection's GPU is refused before any launch."""

import pytest
import torch

from sushi_b200 import Codebook, Decode, Exl3Error, Proj, exl3
from test_kv4_arguments import OnGpu


@pytest.mark.parametrize("elsewhere", [-1, 1])
def test_an_out_elsewhere_is_refused(monkeypatch, elsewhere):
    calls = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    monkeypatch.setattr(exl3, "lib", lambda: Library())
    monkeypatch.setattr(exl3, "_stream", lambda: 7)
    half = lambda *s: OnGpu(torch.ones(s, dtype=torch.float16))
    proj = Proj(OnGpu(torch.zeros((1, 8, 8, 32), dtype=torch.int16)), half(1, 128), half(1, 128))
    x, out = half(2, 128), torch.zeros((2, 128), dtype=torch.float16)
    exl3.linear(x, proj, Decode(Codebook.MCG), out=OnGpu(out))
    assert calls == ["sx_linear"]
    with pytest.raises(Exl3Error, match="SX_ERR_BAD_SHAPE"):
        exl3.linear(x, proj, Decode(Codebook.MCG), out=OnGpu(out, elsewhere))
    assert calls == ["sx_linear"]
