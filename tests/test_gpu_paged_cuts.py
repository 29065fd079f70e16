"""The decode attention's parts: every least number of units, from positions cut as finely as they can be to items left whole; values
of the knob that make no sense count as one."""
import pytest
import torch

import paged_oracle as PO

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("units", ["-3", "0", "1", "3", "16", "1000"])
@pytest.mark.parametrize("lens", [[(9000, 1), (4095, 1), (0, 1)], [(2000, 4), (31, 3)], [(300, 1)] * 50])
def test_attention_with_parts_of_any_length(monkeypatch, units, lens):
    from turbo_lossless_b200 import Split12Engine
    monkeypatch.setenv("S12_PAGED_FORCE", "1")
    monkeypatch.setenv("S12_PAGED_TEAM", "4")
    monkeypatch.setenv("S12_PAGED_MIN_UNITS", units)
    e = Split12Engine()
    c = PO.Case(lens, 8, 2, 128, 64, seed=131)
    ws = e.attention_paged_workspace(8, 2, 128, len(lens), c.max_new)
    want, bound = PO.attention(c, 0.1)
    for _ in range(3):
        out = torch.zeros(c.tokens, 8 * 128, dtype=torch.int16, device="cuda")
        e.attention_paged(c.q, *c.cache(), out, c.table, c.kv_len, c.q_start, 8, 0.1, c.max_new, c.max_len, ws)
        torch.cuda.synchronize()
        assert ((out.view(torch.bfloat16).double() - want).abs() <= bound).all()
    assert e.device_status() == 0
