"""Scales of a paged cache that differ by many binary orders: a row keeps the digits of what it sees, whatever the scales of
positions that it does not see, or that its weights make nothing of.

The bound counts roundings over the positions that a row sees alone (p: weights over the row's largest, z = p times the value's
scale, n: positions seen):
  the output to bf16: 2^-8 of the value;
  q, k to f16, or q to 15 bits of its largest, or none of these: a score is off by d = scale * ((2 * 2^-11 + 2^-14) sum |q||k| +
    2^-15 max|q| sum |k|), 2^-14 for scales that are a sum of two f16; a weight by e^(2d) - 1 of itself, numerator and sum alike;
  a weight, a value's scale and their product to f16: 3 * 2^-11 of |p v|; below f16's normal numbers 2^-32 for each weight, or
    2^-31 of the largest z for each z (a row's unit keeps that one at 2^6 or more);
  z to 15 bits of the largest of 32 neighbours: 2^-15 of that largest for each of the 32 (the position's code is at most 127);
  sums in 32 bits: 2^-20 of the sum of magnitudes."""
import math

import pytest
import torch

import paged_oracle as PO

pytestmark = pytest.mark.gpu

KERNELS = {"rule": ("0", "0"), "digits": ("1", "4"), "warps": ("1", "1"), "tiles": ("2", "0")}


def attention(c, scale, absent=()):
    """(out, bound) in 64 bits; the rows that see a scale that is not finite are NaN."""
    hd, gqa = c.hd, c.n_head // c.n_kv
    out = torch.zeros(c.tokens, c.n_head * hd, dtype=torch.float64, device=c.q.device)
    bound, row = torch.zeros_like(out), 0
    for i, (before, new) in enumerate(c.lens):
        n, dev = before + new, c.q.device
        if new == 0:
            continue
        t = torch.arange(n, device=dev)
        keep = torch.ones(n, dtype=torch.bool, device=dev)
        for s, p in absent:
            if s == i:
                keep &= t // c.page != p
        page, slot = c.table[i].long()[t // c.page].clamp(0, c.codes[0].shape[0] - 1), t % c.page
        seen = (t[None] <= torch.arange(before, n, device=dev)[:, None]) & keep[None]
        for h in range(c.n_head):
            sk, sv = (x[page, h // gqa, slot].double() for x in c.scales)
            sk, sv = torch.where(keep, sk, 0), torch.where(keep, sv, 0)
            k, v = c.codes[0][page, h // gqa, slot].double() * sk[:, None], c.codes[1][page, h // gqa, slot].double() * sv[:, None]
            q = c.q[row:row + new, h * hd:(h + 1) * hd].double()
            s = torch.where(seen, q @ k.nan_to_num(0).T * scale, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, 0, m))
            den = p.sum(1, keepdim=True)
            den = torch.where(den == 0, 1, den)
            size, o = p @ v.abs().nan_to_num(0) / den, p @ v.nan_to_num(0) / den
            d = scale * ((2.0 ** -10 + 2.0 ** -14) * q.abs() @ k.abs().nan_to_num(0).T + 2.0 ** -15 * q.abs().amax(1, keepdim=True) * k.abs().nan_to_num(0).sum(1)[None])
            d = torch.where(seen, d, 0).amax(1, keepdim=True)
            z = torch.where(seen, p * sv.abs().nan_to_num(0), 0)
            chunks = torch.nn.functional.pad(z, (0, -n % 32)).view(new, -(-n // 32), 32).amax(2).sum(1, keepdim=True)
            small = 2.0 ** -32 * (seen.double() @ v.abs().nan_to_num(0)) + 2.0 ** -31 * 127 * seen.sum(1, keepdim=True) * z.amax(1, keepdim=True)
            err = size * (torch.expm1(2 * d) + 3 * 2.0 ** -11 + 2.0 ** -20) + (32 * 2.0 ** -15 * 127 * chunks + small) / den
            odd = (seen & ~(sk + sv).isfinite()[None]).any(1)
            o[odd] = math.nan
            out[row:row + new, h * hd:(h + 1) * hd] = o
            bound[row:row + new, h * hd:(h + 1) * hd] = (2.0 ** -8 * (o.abs() + err) + err).nan_to_num(math.inf)
        row += new
    return out, bound


def run(c, scale, kernel, monkeypatch):
    from turbo_lossless_b200 import Split12Engine
    monkeypatch.setenv("S12_PAGED_FORCE", KERNELS[kernel][0])
    monkeypatch.setenv("S12_PAGED_TEAM", KERNELS[kernel][1])
    e = Split12Engine()
    out = torch.zeros(c.tokens, c.n_head * c.hd, dtype=torch.int16, device="cuda")
    e.attention_paged(c.q, *c.cache(), out, c.table, c.kv_len, c.q_start, c.n_head, scale, c.max_new, c.max_len)
    torch.cuda.synchronize()
    return out.view(torch.bfloat16).double(), e.device_status()


def check(got, want, bound):
    assert torch.equal(got.isnan(), want.isnan())
    over = torch.where(want.isnan(), 0, (got - want).abs() - bound)
    assert over.max().item() <= 0, f"{over.max().item()} above the bound, {int((over > 0).sum())} elements"


def scales_of(c, seq, which):
    """(read, write) of the scales [position][kv head] of a sequence."""
    n = sum(c.lens[seq])
    t = torch.arange(n, device="cuda")
    page, slot = c.table[seq].long()[t // c.page], t % c.page

    def write(x):
        c.scales[which][page, :, slot] = x
    return c.scales[which][page, :, slot], write


@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 2, 128), (4, 2, 64), (3, 1, 96), (2, 2, 80)])
@pytest.mark.parametrize("orders", [10, 14, 18, 24, 40, 60])
@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_values_before_one_of_a_far_larger_scale(monkeypatch, kernel, orders, n_head, n_kv, hd):
    """A causal row does not see a later position: not its scale either.  In the first tile, in a later one, and in all of them."""
    for lens, at in (([(0, 200)], [100]), ([(0, 200)], [3]), ([(0, 420)], [330]), ([(100, 200)], [120, 260])):
        c = PO.Case(lens, n_head, n_kv, hd, 32, seed=101)
        old, write = scales_of(c, 0, 1)
        old[at] *= 2.0 ** orders
        write(old * 2.0 ** -20)
        got, status = run(c, hd ** -0.5, kernel, monkeypatch)
        assert status == 0
        check(got, *attention(c, hd ** -0.5))


@pytest.mark.parametrize("kernel", sorted(KERNELS))
@pytest.mark.parametrize("spread", [3, 9, 30, 70])
@pytest.mark.parametrize("lens", [[(0, 300), (700, 150)], [(3000, 260)]])
def test_values_of_scales_all_over(monkeypatch, kernel, spread, lens):
    """Scales over 2 * spread binary orders, zeros among them, from position to position."""
    c = PO.Case(lens, 8, 2, 128, 64, seed=102)
    g = torch.Generator().manual_seed(spread)
    for i, (b, n) in enumerate(lens):
        old, write = scales_of(c, i, 1)
        turn = torch.exp2((torch.rand(b + n, 2, generator=g) * 2 - 1) * spread)
        turn[torch.rand(b + n, 2, generator=g) < 0.1] = 0
        write(old * turn.cuda())
    got, status = run(c, 0.09, kernel, monkeypatch)
    assert status == 0
    check(got, *attention(c, 0.09))


@pytest.mark.parametrize("kernel", sorted(KERNELS))
@pytest.mark.parametrize("orders", [-60, -25, 25, 60])
def test_large_values_whose_weight_is_nothing(monkeypatch, kernel, orders):
    """The first half's values are 2^orders of the second's, and its scores so far below that its weights are 2^-150 (no score of
    the case needs more than 16 bits): the sums keep the digits of the second half, and a row of the first half its own."""
    c = PO.Case([(0, 500)], 4, 2, 128, 64, seed=103)
    old, write = scales_of(c, 0, 1)
    old[:250] *= 2.0 ** orders
    write(old)
    # scores: one large dim of q against codes that say which half it is
    c.q[:, ::128] = 64.0
    t = torch.arange(500, device="cuda")
    page, slot = c.table[0].long()[t // 64], t % 64
    c.codes[0][page, :, slot, 0] = torch.where(t < 250, -100, 100).to(torch.int8)[:, None]
    sk, write_k = scales_of(c, 0, 0)
    write_k(torch.full_like(sk, 2.0 ** -6))
    c.q.mul_(0.5)
    got, status = run(c, 1.0, kernel, monkeypatch)
    assert status == 0
    check(got, *attention(c, 1.0))


@pytest.mark.parametrize("kernel", sorted(KERNELS))
@pytest.mark.parametrize("orders", [12, 20, 30, 40])
@pytest.mark.parametrize("hd", [128, 64])
def test_keys_before_one_of_a_far_larger_scale(monkeypatch, kernel, orders, hd):
    """Rows that do not see the key of the large scale keep the digits of theirs; those that see it have a score of 2^orders."""
    for lens, at in (([(0, 200)], 150), ([(0, 300)], 299), ([(120, 90)], 170)):
        c = PO.Case(lens, 8, 2, hd, 64, seed=104)
        old, write = scales_of(c, 0, 0)
        old[at] *= 2.0 ** orders
        write(old)
        got, status = run(c, hd ** -0.5, kernel, monkeypatch)
        assert status == 0
        check(got, *attention(c, hd ** -0.5))


@pytest.mark.parametrize("kernel", sorted(KERNELS))
@pytest.mark.parametrize("which", [0, 1])
def test_far_scales_next_to_missing_pages_and_nans(monkeypatch, kernel, which):
    """A page that the table lacks, and a scale that is not finite, in a sequence whose values span 2^40."""
    for bad in (math.nan, math.inf)[:1 + which]:                      # a key's infinite scale gives a NaN or an infinite score
        c = PO.Case([(0, 310), (40, 60)], 8, 2, 128, 32, seed=105)
        old, write = scales_of(c, 0, 1)
        old[::7] *= 2.0 ** 40
        write(old)
        old, write = scales_of(c, 0, which)
        old[200, 1] = bad
        write(old)
        want = attention(c, 0.1, absent=[(0, 2), (0, 5)])
        c.table[0, 2], c.table[0, 5] = -1, c.codes[0].shape[0]
        got, status = run(c, 0.1, kernel, monkeypatch)
        assert status == 0x100000
        check(got, *want)


def test_wide_and_ordinary_sequences_in_one_call(monkeypatch):
    """More items than resident CTAs, every third of them wide from somewhere on; the same bits every time."""
    lens = [(i * 37 % 211 if (i * i + 3 * i) % 97 else 0, (i * i + 3 * i) % 97) for i in range(200)] + [(0, 700), (900, 3), (0, 1), (300, 400)]
    c = PO.Case(lens, 8, 4, 128, 32, seed=106)
    for i, (b, n) in enumerate(lens):
        if n and i % 3 == 0:
            old, write = scales_of(c, i, 1)
            old[(b + n) * 2 // 3] *= 2.0 ** 30
            write(old)
    first, status = run(c, 0.09, "tiles", monkeypatch)
    assert status == 0
    check(first, *attention(c, 0.09))
    for _ in range(10):
        again, status = run(c, 0.09, "tiles", monkeypatch)
        assert status == 0 and torch.equal(again, first)


@pytest.mark.parametrize("spread", [0.4, 12])
def test_a_long_prompt(monkeypatch, spread):
    """20 000 positions: running sums over them in 32 bits, two heads, a chunk of rows at the end and at the start."""
    c = PO.Case([(20000, 130), (0, 130)], 2, 1, 64, 128, seed=107)
    g = torch.Generator().manual_seed(7)
    old, write = scales_of(c, 0, 1)
    write(old * torch.exp2(torch.randn(20130, 1, generator=g) * spread / 2).cuda())
    for kernel in ("tiles", "digits"):
        got, status = run(c, 0.125, kernel, monkeypatch)
        assert status == 0
        check(got, *attention(c, 0.125))
