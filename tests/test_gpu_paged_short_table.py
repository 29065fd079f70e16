"""A block table with fewer pages than a sequence's positions need: these are masked, and the status word says so."""
import pytest

import paged_oracle as PO

pytestmark = pytest.mark.gpu

KERNELS = {"rule": ("0", "0"), "digits": ("1", "4"), "warps": ("1", "1"), "tiles": ("2", "0")}


@pytest.mark.parametrize("kernel", sorted(KERNELS))
@pytest.mark.parametrize("hd", [128, 64, 96, 80])
@pytest.mark.parametrize("lens", [[(300, 1), (20, 1)], [(255, 1)], [(100, 200), (20, 30)], [(250, 10)], [(0, 600)]])
def test_positions_past_the_table(monkeypatch, kernel, hd, lens):
    import torch
    from turbo_lossless_b200 import Split12Engine
    monkeypatch.setenv("S12_PAGED_FORCE", KERNELS[kernel][0])
    monkeypatch.setenv("S12_PAGED_TEAM", KERNELS[kernel][1])
    e = Split12Engine()
    c = PO.Case(lens, 8, 2, hd, 64, seed=111)
    pages = -(-int(c.kv_len.max()) // 64)
    short = pages - 1
    want = PO.attention(c, 0.1, absent=[(i, p) for i in range(len(lens)) for p in range(short, pages)])

    def run(table_pages, max_len):
        out = torch.zeros(c.tokens, 8 * hd, dtype=torch.int16, device="cuda")
        e.attention_paged(c.q, *c.cache(), out, c.table[:, :table_pages], c.kv_len, c.q_start, 8, 0.1, c.max_new, max_len)
        torch.cuda.synchronize()
        return out.view(torch.bfloat16).double(), e.device_status()

    got, status = run(short, c.max_len)
    assert status == 0x100000 and ((got - want[0]).abs() <= want[1]).all()
    got, status = run(short, 64 * short)                              # the caller's bound masks them: nothing is missing
    assert status == 0 and ((got - want[0]).abs() <= want[1]).all()
    got, status = run(pages, c.max_len)
    assert status == 0
