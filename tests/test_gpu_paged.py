"""The paged INT8 cache's operators against 64 bits (paged_oracle.py derives the bounds)."""
import math

import pytest
import torch

import paged_oracle as PO

pytestmark = pytest.mark.gpu

KINDS = {
    "one_token": [(0, 1)],
    "decode": [(n - 1, 1) for n in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 200, 1000)],
    "long_decode": [(9000, 1), (4095, 1), (0, 1)],
    "few_tokens": [(500, 4), (0, 3), (90, 1), (33, 0), (1000, 4), (0, 1), (2, 2)],
    "two_tokens_far": [(6000, 2), (5, 2)],
    "prompt": [(0, 150)],
    "tile_ends": [(0, n) for n in (31, 32, 33, 63, 64, 65)] + [(0, n) for n in (127, 128, 129)],
    "ragged": [(0, 7), (0, 0), (130, 5), (0, 1), (3, 261), (0, 0)],
    "chunks": [(1000, 3), (64, 64), (77, 200)],
}
SHAPES = [(32, 8, 128), (8, 8, 128), (8, 1, 128), (6, 2, 128), (10, 2, 64), (16, 1, 96), (4, 2, 64), (40, 2, 128), (2, 2, 20), (4, 2, 80), (2, 1, 256)]


@pytest.fixture(params=["rule", "digits", "warps", "tiles"])
def kernel(request, monkeypatch):
    """The kernel that the rule chooses, and each of the two for heads of 64, 96 and 128 whatever the rule says, the first with
    four warps to a part and with one to an item."""
    monkeypatch.setenv("S12_PAGED_FORCE", {"rule": "0", "digits": "1", "warps": "1", "tiles": "2"}[request.param])
    monkeypatch.setenv("S12_PAGED_TEAM", {"rule": "0", "digits": "4", "warps": "1", "tiles": "0"}[request.param])
    return request.param


def run_attention(c, scale, q=None, out=None, workspace=None, table=None):
    from turbo_lossless_b200 import Split12Engine
    e = Split12Engine()
    if out is None:
        out = torch.full((c.q.shape[0], c.n_head * c.hd), 0x5A5A, dtype=torch.int16, device="cuda")
    q_start = None if all(n == 1 for _, n in c.lens) and c.q.shape[0] == c.tokens else c.q_start
    e.attention_paged(c.q if q is None else q, *c.cache(), out, c.table if table is None else table, c.kv_len, q_start, c.n_head, scale,
                      c.max_new, c.max_len, workspace)
    torch.cuda.synchronize()
    return out, e.device_status()


def check(out, want, bound):
    got = out.view(torch.bfloat16).double()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, f"{over} above the bound"


@pytest.mark.parametrize("n_head,n_kv,hd", SHAPES)
@pytest.mark.parametrize("kind", sorted(KINDS))
def test_attention_against_64_bits(kernel, kind, n_head, n_kv, hd):
    if kernel != "rule" and hd not in (64, 96, 128):
        pytest.skip("other heads have one kernel")
    page = 16 << (len(kind) + n_head) % 4
    c = PO.Case(KINDS[kind], n_head, n_kv, hd, page, seed=7)
    out, status = run_attention(c, hd ** -0.5)
    assert status == 0
    check(out, *PO.attention(c, hd ** -0.5))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_attention_over_every_page_size(kernel, page):
    for lens in ([(0, 300), (500, 40)], [(700, 1), (31, 1), (1023, 1)]):
        c = PO.Case(lens, 16, 4, 128, page, seed=page)
        out, status = run_attention(c, 0.1)
        assert status == 0
        check(out, *PO.attention(c, 0.1))


@pytest.mark.parametrize("lens", [[(5, 1), (90, 1)], [(5, 30), (90, 170)]])
def test_rows_with_strides_and_rows_behind_the_last_sequence(kernel, lens):
    c = PO.Case(lens, 8, 2, 128, 32, seed=1, spare_rows=9)
    wide = torch.full((c.q.shape[0], c.q.shape[1] + 24), math.nan, device="cuda")
    wide[:, :c.q.shape[1]] = c.q
    wide[c.tokens:] = math.nan
    out = torch.full((c.q.shape[0], c.q.shape[1] + 40), 77, dtype=torch.int16, device="cuda")
    run_attention(c, 0.09, q=wide[:, :c.q.shape[1]], out=out[:, :c.q.shape[1]])
    check(out[:c.tokens, :c.q.shape[1]].contiguous(), *PO.attention(c, 0.09))
    assert (out[c.tokens:] == 77).all() and (out[:, c.q.shape[1]:] == 77).all()


@pytest.mark.parametrize("hd", [128, 80])
@pytest.mark.parametrize("lens", [[(200, 1), (70, 1)], [(100, 100), (70, 3)]])
def test_sequences_that_hold_nothing_give_zeros(kernel, lens, hd):
    c = PO.Case(lens + [(0, lens[0][1])], 8, 2, hd, 16, seed=2)
    c.kv_len[2] = 0                                                   # its tokens come before position 0
    out, status = run_attention(c, 0.1)
    assert status == 0
    n = c.tokens - lens[0][1]
    assert (out[n:] == 0).all()
    c.lens = c.lens[:2]
    c.tokens = n
    check(out[:n], *PO.attention(c, 0.1))


@pytest.mark.parametrize("hd", [128, 80])
@pytest.mark.parametrize("lens", [[(400, 1), (70, 1)], [(200, 100), (70, 3)]])
def test_pages_that_the_table_lacks_are_masked_and_reported(kernel, lens, hd):
    c = PO.Case(lens, 8, 2, hd, 64, seed=3)
    want = PO.attention(c, 0.1, absent=[(0, 1), (0, 3), (1, 0)])
    c.table[0, 1], c.table[0, 3], c.table[1, 0] = -1, c.codes[0].shape[0], 1 << 30
    out, status = run_attention(c, 0.1)
    assert status == 0x100000
    check(out, *want)


@pytest.mark.parametrize("lens", [[(300, 1)], [(100, 200)]])
def test_sizes_of_values_and_scores(kernel, lens):
    """Scales over 30 binary orders, one score far above the others, q of a row with one large element."""
    c = PO.Case(lens, 8, 2, 128, 64, seed=4)
    t = torch.arange(sum(lens[0]), device="cuda")
    c.scales[1][c.table[0].long()[t // 64], :, t % 64] *= torch.exp2((t % 31 - 15).float())[:, None]
    c.q[:, 5] *= 40
    c.codes[0][c.table[0, 0].long(), :, 3] = 127
    out, _ = run_attention(c, 0.1)
    check(out, *PO.attention(c, 0.1))


@pytest.mark.parametrize("lens", [[(300, 1), (20, 1)], [(100, 200), (20, 30)]])
@pytest.mark.parametrize("what", ["q", "scale_k", "scale_v"])
def test_a_nan_stays_with_the_rows_that_use_it(kernel, lens, what):
    c = PO.Case(lens, 8, 2, 128, 32, seed=5)
    want, bound = PO.attention(c, 0.1)
    if what == "q":
        c.q[0, 2 * 128 + 3] = math.nan
        hit = [(0, 2)]
    else:
        c.scales[what == "scale_v"][c.table[0, 0].long(), 1, 9] = math.nan
        hit = [(r, h) for r in range(lens[0][1]) for h in range(4, 8)]
    out, _ = run_attention(c, 0.1)
    got = out.view(torch.bfloat16).double().view(c.tokens, 8, 128)
    touched = torch.zeros(c.tokens, 8, dtype=torch.bool, device="cuda")
    for r, h in hit:
        touched[r, h] = True
    assert torch.isnan(got[touched]).any(-1).all()
    check(out.view(c.tokens, 8, 128)[~touched], want.view(c.tokens, 8, 128)[~touched], bound.view(c.tokens, 8, 128)[~touched])


@pytest.mark.parametrize("lens", [[(300, 1), (20, 1), (4000, 1)], [(100, 200), (20, 30)]])
def test_a_captured_call_follows_the_lengths_and_repeats_its_bits(kernel, lens):
    from turbo_lossless_b200 import Split12Engine
    c = PO.Case(lens, 16, 4, 128, 64, seed=6)
    e = Split12Engine()
    out = torch.zeros(c.tokens, 16 * 128, dtype=torch.int16, device="cuda")
    ws = e.attention_paged_workspace(16, 4, 128, len(lens), c.max_new)
    q_start = None if c.max_new == 1 else c.q_start
    args = (c.q, *c.cache(), out, c.table, c.kv_len, q_start, 16, 0.1, c.max_new, c.max_len, ws)
    e.attention_paged(*args)
    torch.cuda.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        e.attention_paged(*args)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    c.lens = [(b // 2, n) for b, n in lens]
    c.kv_len.copy_(torch.tensor([b + n for b, n in c.lens], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(out, *PO.attention(c, 0.1))


STORES = [("decode", 32, 8, 128), ("ragged", 6, 2, 128), ("prompt", 4, 4, 64), ("tile_ends", 16, 1, 96), ("chunks", 2, 2, 20), ("chunks", 3, 1, 256),
          ("long_decode", 8, 1, 80), ("one_token", 32, 8, 128)]


@pytest.mark.parametrize("kind,n_head,n_kv,hd", STORES)
def test_store_against_64_bits(kind, n_head, n_kv, hd):
    """Codes and scales are the exact ones; q is off by the rounding of cos, sin, two products and a sum: 5 * 2^-24 of the
    pair's size."""
    from turbo_lossless_b200 import Split12Engine
    c = PO.Case(KINDS[kind], n_head, n_kv, hd, 16 << n_head % 4, seed=11, spare_rows=3)
    c.k[:c.tokens // 2, :hd] *= 1000
    c.v[0] = 0
    q, k, v = c.q.clone(), c.k.clone(), c.v.clone()
    want_q, codes, scales = PO.store(c, 500000.0)
    e = Split12Engine()
    e.rope_store_kv_paged(c.q, c.k, c.v, *c.cache(), c.table, c.kv_len, c.q_start, n_head, 500000.0)
    torch.cuda.synchronize()
    assert e.device_status() == 0
    assert torch.equal(c.k, k) and torch.equal(c.v, v) and torch.equal(c.q[c.tokens:], q[c.tokens:])
    pair = q[:c.tokens].double().view(c.tokens, n_head, 2, hd // 2)
    size = (pair[:, :, 0].square() + pair[:, :, 1].square()).sqrt().repeat(1, 1, 2).view(c.tokens, -1)
    assert ((c.q[:c.tokens].double() - want_q).abs() <= 5 * 2.0 ** -24 * math.sqrt(2) * size).all()
    for j in (0, 1):
        assert torch.equal(c.codes[j], codes[j])
        assert torch.equal(c.scales[j].nan_to_num(-1), scales[j].nan_to_num(-1))


def test_store_keeps_other_buffers_and_reports_missing_pages():
    from turbo_lossless_b200 import Split12Engine
    c = PO.Case([(10, 60), (0, 5), (3, 2)], 8, 2, 64, 16, seed=12)
    c.table[0, 2] = -1
    c.table[1, 0] = c.codes[0].shape[0]
    c.kv_len[2] = 0                                                   # rows that hold no sequence: no error, no store
    want_q, codes, scales = PO.store(c.__class__([(10, 60), (0, 5), (3, 2)], 8, 2, 64, 16, seed=12), 10000.0)
    fused = torch.zeros(c.tokens, 8 * 64 + 4 * 64, device="cuda")     # q, k, v side by side, as one projection gives them
    fused[:, :512], fused[:, 512:640], fused[:, 640:] = c.q, c.k, c.v
    before = [x.clone() for x in c.cache()]
    keep, q_out = fused.clone(), torch.zeros(c.tokens, 512, device="cuda")
    e = Split12Engine()
    e.rope_store_kv_paged(fused[:, :512], fused[:, 512:640], fused[:, 640:], *c.cache(), c.table, c.kv_len, c.q_start, 8, 10000.0, q_out=q_out)
    torch.cuda.synchronize()
    assert e.device_status() == 0x100000 and torch.equal(fused, keep)
    for x, b, w in zip(c.cache(), before, (*codes, *scales)):
        for t in range(10, 70):
            page = int(c.table[0, t // 16])
            if page >= 0:
                assert torch.equal(x[page, :, t % 16], w[page, :, t % 16])
                b[page, :, t % 16] = x[page, :, t % 16]
        assert torch.equal(x.nan_to_num(-1), b.nan_to_num(-1)) if x.is_floating_point() else torch.equal(x, b)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_value_that_is_not_finite_marks_its_row(bad):
    from turbo_lossless_b200 import Split12Engine
    c = PO.Case([(0, 4)], 4, 2, 128, 16, seed=13)
    _, _, scales = PO.store(c, 10000.0)
    c.k[1, 7], c.v[2, 128 + 5] = bad, bad
    Split12Engine().rope_store_kv_paged(c.q, c.k, c.v, *c.cache(), c.table, c.kv_len, c.q_start, 4, 10000.0)
    page = c.table[0, 0].long()
    for j, row, head in ((0, 1, 0), (1, 2, 1)):
        got, want = c.scales[j][page, :, :4].clone(), scales[j][page, :, :4].clone()
        assert not torch.isfinite(got[head, row])
        got[head, row] = want[head, row] = 0
        assert torch.equal(got, want)


@pytest.mark.parametrize("layers,pages,n_kv,page,hd,count", [(1, 5, 1, 16, 4, 1), (3, 40, 2, 32, 96, 17), (2, 9, 8, 64, 128, 4), (5, 7, 3, 16, 20, 2), (1, 300, 1, 16, 64, 150)])
def test_copy_pages(layers, pages, n_kv, page, hd, count):
    from turbo_lossless_b200 import Split12Engine
    g = torch.Generator(device="cuda").manual_seed(count)
    shape = (layers, pages, n_kv, page)
    kv = [torch.randint(-128, 128, (*shape, hd), dtype=torch.int8, device="cuda", generator=g) for _ in "kv"]
    sc = [torch.randn(shape, device="cuda", generator=g) for _ in "kv"]
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    src, dst = order[:count].clone(), order[count:2 * count].clone()
    want = [x.clone() for x in (*kv, *sc)]
    status = 0
    if count > 3:
        src[1] = src[0]                                               # one source twice
    for i in range(count):
        if count > 3 and i == 2:                                      # one copy that is skipped
            src[i], status = pages, 0x100000
            continue
        for x in want:
            x[:, dst[i]] = x[:, src[i]]
    e = Split12Engine()
    e.copy_pages(*kv, *sc, src, dst)
    torch.cuda.synchronize()
    assert e.device_status() == status
    for x, w in zip((*kv, *sc), want):
        assert torch.equal(x, w)
    e.copy_pages(*kv, *sc, src[:0], dst[:0])                          # nothing to do


def test_wrappers_refuse_what_the_kernels_cannot_take():
    from turbo_lossless_b200 import S12Error, Split12Engine
    c = PO.Case([(0, 4), (3, 2)], 4, 2, 128, 16, seed=14)
    e = Split12Engine()
    out = torch.zeros(c.tokens, 512, dtype=torch.int16, device="cuda")
    ok = dict(q=c.q, kv_k=c.codes[0], kv_v=c.codes[1], scale_k=c.scales[0], scale_v=c.scales[1], out_bf16=out, block_table=c.table,
              kv_len=c.kv_len, q_start=c.q_start, n_head=4, scale=0.1, max_new=4, max_len=5)
    e.attention_paged(**ok)
    for edit in (dict(q=c.q.double()), dict(q=c.q[:, :500]), dict(q=c.q.t()), dict(q=c.q.cpu()), dict(kv_k=c.codes[0].cpu()), dict(kv_v=c.codes[1][1:]),
                 dict(scale_k=c.scales[0].double()), dict(kv_k=c.codes[0].transpose(1, 2), kv_v=c.codes[1].transpose(1, 2)), dict(out_bf16=out[:3]),
                 dict(out_bf16=out.view(torch.bfloat16)), dict(block_table=c.table.long()), dict(block_table=c.table[:1]), dict(kv_len=c.kv_len.cpu()),
                 dict(q_start=c.q_start[:2]), dict(q_start=c.q_start.long()), dict(block_table=c.table.t().contiguous().t())):
        with pytest.raises(ValueError):
            e.attention_paged(**{**ok, **edit})
    for edit in (dict(q_start=None), dict(n_head=3), dict(max_new=0), dict(max_len=0), dict(n_head=0)):
        with pytest.raises(S12Error):
            e.attention_paged(**{**ok, **edit})


def test_pages_beyond_32_bit_offsets():
    """A pool of 4.6 GB for K and V each, of which the sequences hold the last pages: every path reads and writes there."""
    from turbo_lossless_b200 import Split12Engine
    e, pages = Split12Engine(), 70000
    pool = [torch.empty(pages, 8, 64, 128, dtype=torch.int8, device="cuda") for _ in "kv"] + [torch.empty(pages, 8, 64, device="cuda") for _ in "kv"]
    for lens in ([(130, 1), (64, 1)], [(70, 80), (0, 9)]):
        c = PO.Case(lens, 16, 8, 128, 64, seed=21)
        small = c.codes[0].shape[0]
        for x, y in zip(pool, c.cache()):
            x[pages - small:] = y
        table = torch.where(c.table >= 0, c.table + (pages - small), -1)
        q_start = None if c.max_new == 1 else c.q_start
        _, codes, scales = PO.store(c, 10000.0)
        e.rope_store_kv_paged(c.q, c.k, c.v, *pool, table, c.kv_len, q_start, 16, 10000.0)
        for x, y in zip(pool, (*codes, *scales)):
            assert torch.equal(x[pages - small:].nan_to_num(-1), y.nan_to_num(-1)) if x.is_floating_point() else torch.equal(x[pages - small:], y)
        c.codes, c.scales = codes, scales
        out = torch.zeros(c.tokens, 16 * 128, dtype=torch.int16, device="cuda")
        e.attention_paged(c.q, *pool, out, table, c.kv_len, q_start, 16, 0.1, c.max_new, c.max_len)
        check(out, *PO.attention(c, 0.1))
        src, dst = table[0, :2].clone(), torch.tensor([1, 0], dtype=torch.int32, device="cuda")
        e.copy_pages(*pool, src, dst)
        assert all(torch.equal(x[dst.long()].nan_to_num(-1) if x.is_floating_point() else x[dst.long()], x[src.long()].nan_to_num(-1) if x.is_floating_point() else x[src.long()]) for x in pool)
    assert e.device_status() == 0


def test_one_workspace_serves_calls_of_other_sizes_in_turn():
    """The workspace is as it was after every call: whatever came before, a call's bits are the same."""
    from turbo_lossless_b200 import Split12Engine
    e = Split12Engine()
    shapes = [([(9000, 1), (4095, 1), (0, 1)], 8, 1), ([(300, 1)] * 40, 32, 8), ([(2000, 4), (31, 3)], 16, 2), ([(100000, 1)], 4, 4)]
    cases = [PO.Case(lens, h, hkv, 128, 64, seed=31) for lens, h, hkv in shapes]
    ws = e.attention_paged_workspace(32, 1, 128, 40, 8)
    outs = []
    for turn in range(3):
        for c in cases[::-1] if turn else cases:
            out, status = run_attention(c, 0.1, workspace=ws)
            assert status == 0
            outs.append((c, out))
    for c in cases:
        mine = [o for k, o in outs if k is c]
        assert all(torch.equal(o, mine[0]) for o in mine)
        check(mine[0], *PO.attention(c, 0.1))
    assert not ws.view(torch.int32)[-(32 * 1 * 40 * 2) // 4:].any()


def test_two_streams_with_workspaces_of_their_own():
    from turbo_lossless_b200 import Split12Engine
    e = Split12Engine()
    cases = [PO.Case([(20000 + i, 1), (5, 1)], 8, 1, 128, 64, seed=40 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    spaces = [e.attention_paged_workspace(8, 1, 128, 2, 1) for _ in cases]
    outs = [torch.zeros(2, 8 * 128, dtype=torch.int16, device="cuda") for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st, ws, out in zip(cases, streams, spaces, outs):
            e.attention_paged(c.q, *c.cache(), out, c.table, c.kv_len, None, 8, 0.1, 1, c.max_len, ws, stream=st)
    torch.cuda.synchronize()
    for c, out in zip(cases, outs):
        check(out, *PO.attention(c, 0.1))
    with pytest.raises(ValueError):
        e.attention_paged(cases[0].q, *cases[0].cache(), outs[0], cases[0].table, cases[0].kv_len, None, 8, 0.1, 1, 30000, stream=streams[0])


def test_dependent_launches_wait_for_one_another():
    """Store, attention over what it stored, and a page copy, replayed as a graph of dependent launches."""
    from turbo_lossless_b200 import Split12Engine
    e = Split12Engine()
    for lens in ([(200, 1), (63, 1)], [(64, 100), (0, 40)]):
        c = PO.Case(lens, 8, 2, 128, 64, seed=51)
        q_start = None if c.max_new == 1 else c.q_start
        ws = e.attention_paged_workspace(8, 2, 128, 2, c.max_new)
        q_out, out = torch.zeros_like(c.q), torch.zeros(c.tokens, 8 * 128, dtype=torch.int16, device="cuda")
        src, dst = c.table[0, :1].clone(), torch.tensor([sorted(set(range(c.codes[0].shape[0])) - set(c.table.flatten().tolist()))[0]], dtype=torch.int32, device="cuda")

        def step():
            e.rope_store_kv_paged(c.q, c.k, c.v, *c.cache(), c.table, c.kv_len, q_start, 8, 10000.0, q_out=q_out)
            e.attention_paged(q_out, *c.cache(), out, c.table, c.kv_len, q_start, 8, 0.1, c.max_new, c.max_len, ws)
            e.copy_pages(*c.cache(), src, dst)
        step()
        torch.cuda.synchronize()
        old = e.set_dependent_launch(True)
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                for _ in range(4):
                    step()
        finally:
            e.set_dependent_launch(old)
        for x in (q_out, out):
            x.zero_()
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        q = c.q
        c.q = q_out
        check(out, *PO.attention(c, 0.1))
        c.q = q
        assert torch.equal(c.codes[0][dst.long()], c.codes[0][src.long()]) and e.device_status() == 0


def test_codes_of_values_on_a_border():
    """Values of few bits, many of which lie halfway between two codes: both store kernels (rows on 16-byte boundaries, and others)
    put them where the rounded product with 127 / absmax, to the nearest even code, puts them.  At position 0 k is not turned."""
    from turbo_lossless_b200 import Split12Engine
    e = Split12Engine()
    for n_kv, hd, page in ((4, 128, 64), (2, 20, 16)):
        c = PO.Case([(0, 1)] * 300, n_kv, n_kv, hd, page, seed=61)
        g = torch.Generator().manual_seed(62)
        for name in ("k", "v"):
            x = torch.randint(-127, 128, (c.tokens, n_kv, hd), generator=g).float() / 2
            x[..., 0] = torch.randint(100, 128, (c.tokens, n_kv), generator=g)
            setattr(c, name, (x * torch.randint(1, 50, (c.tokens, n_kv, 1), generator=g)).view(c.tokens, -1).cuda())
        _, codes, scales = PO.store(c, 10000.0)
        e.rope_store_kv_paged(c.q, c.k, c.v, *c.cache(), c.table, c.kv_len, None, n_kv, 10000.0)
        for j in (0, 1):
            assert torch.equal(c.codes[j], codes[j])
            assert torch.equal(c.scales[j].nan_to_num(-1), scales[j].nan_to_num(-1))


@pytest.mark.parametrize("lens", [[(300, 1), (0, 1)], [(100, 200), (20, 30)]])
@pytest.mark.parametrize("hd", [128, 64, 80])
def test_elements_near_the_largest_float(kernel, lens, hd):
    """q up to 2e38 under a scale that makes ordinary scores of it; values up to 3e38 / 350, whose sums stay finite."""
    c = PO.Case(lens, 8, 2, hd, 64, seed=71)
    c.q *= 2e38 / c.q.abs().max()
    c.scales[0] *= 0.2
    c.scales[1] *= 3e38 / 350 / 127 / c.scales[1].nan_to_num(0).max()
    scale = torch.tensor(1.2e-38).item()
    out, status = run_attention(c, scale)
    assert status == 0
    check(out, *PO.attention(c, scale))


def test_one_value_near_the_largest_float(kernel):
    c = PO.Case([(0, 1), (0, 1)], 8, 2, 128, 64, seed=72)
    c.codes[1].copy_(c.codes[1] % 2)
    c.scales[1] /= c.scales[1].nan_to_num(0).max()
    c.scales[1] *= 3e38
    out, _ = run_attention(c, 0.1)
    check(out, *PO.attention(c, 0.1))


@pytest.mark.parametrize("lens", [[(300, 1), (40, 1)], [(100, 200), (20, 30)]])
@pytest.mark.parametrize("hd", [128, 80])
@pytest.mark.parametrize("size", [1e3, 3e5, -7e6, 1e15, -1e16])
def test_scores_of_any_size(kernel, lens, hd, size):
    """All keys alike: equal scores, however large, are equal weights, as those of q = 0."""
    c = PO.Case(lens, 8, 2, hd, 64, seed=73)
    c.codes[0][:] = c.codes[0][0, :, :1].clone()
    c.scales[0].copy_(torch.where(c.scales[0].isnan(), c.scales[0], abs(size)))
    q = c.q * size
    c.q.zero_()
    want = PO.attention(c, 0.1)
    out, _ = run_attention(c, 0.1, q=q)
    check(out, *want)


@pytest.mark.parametrize("many", [90, 700])
def test_many_sequences_one_of_them_long(kernel, many):
    """Every team looks at all lengths: several to a lane, more than 32 lanes' worth, and a length array off its boundary."""
    if kernel == "tiles" and many > 100:
        pytest.skip("one launch of the other kernel is like any other")
    lens = [(i * 7 % 60, 1) for i in range(many)]
    lens[many * 2 // 3] = (5000, 1)
    c = PO.Case(lens, 4, 1, 64, 32, seed=81)
    for off in (0, 1):
        room = torch.zeros(many + 4, dtype=torch.int32, device="cuda")
        room[off:off + many] = c.kv_len
        c.kv_len = room[off:off + many]
        out, status = run_attention(c, 0.125)
        assert status == 0
        if off == 0:
            want = PO.attention(c, 0.125)
        check(out, *want)


@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 4, 128), (24, 2, 64), (8, 4, 96)])
def test_many_prompts_of_all_lengths(monkeypatch, n_head, n_kv, hd):
    """More tiles of rows than the GPU holds at once, so that a CTA takes one after the other: one or two tiles of rows, an odd or
    an even number of steps, sequences without tokens between them; the same bits every time."""
    monkeypatch.setenv("S12_PAGED_FORCE", "2")
    lens = [(i * 37 % 211, (i * i + 3 * i) % 97) for i in range(330)] + [(0, 400), (900, 3), (0, 1)]
    lens = [(0 if n == 0 else b, n) for b, n in lens]
    c = PO.Case(lens, n_head, n_kv, hd, 32, seed=91)
    first, status = run_attention(c, 0.09)
    assert status == 0
    check(first, *PO.attention(c, 0.09))
    for _ in range(20):
        out, status = run_attention(c, 0.09)
        assert status == 0 and torch.equal(out, first)


def test_many_prompts_in_dependent_launches(monkeypatch):
    """CTAs that take over others' work, and launches that begin while they run."""
    from turbo_lossless_b200 import Split12Engine
    monkeypatch.setenv("S12_PAGED_FORCE", "2")
    e = Split12Engine()
    c = PO.Case([(i * 5 % 90, 1 + i * 29 % 150) for i in range(120)], 8, 4, 128, 32, seed=95)
    ws = e.attention_paged_workspace(8, 4, 128, 120, c.max_new)
    q_out, out = torch.zeros_like(c.q), torch.zeros(c.tokens, 8 * 128, dtype=torch.int16, device="cuda")

    def step():
        e.rope_store_kv_paged(c.q, c.k, c.v, *c.cache(), c.table, c.kv_len, c.q_start, 8, 10000.0, q_out=q_out)
        e.attention_paged(q_out, *c.cache(), out, c.table, c.kv_len, c.q_start, 8, 0.1, c.max_new, c.max_len, ws)
    step()
    torch.cuda.synchronize()
    old = e.set_dependent_launch(True)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(6):
                step()
    finally:
        e.set_dependent_launch(old)
    q_out.zero_()
    out.zero_()
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert e.device_status() == 0
    c.q = q_out
    check(out, *PO.attention(c, 0.1))
