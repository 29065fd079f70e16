"""The paged cache's operators in 64 bits, written from their formulas (test infrastructure)."""
import math

import torch


class Case:
    """Sequences with ``before`` cached and ``new`` packed tokens each over one layer's pages, in shuffled order.

    Scales of rows that no sequence holds, and of positions behind a sequence's end, are NaN: nobody may use them."""

    def __init__(self, lens, n_head, n_kv, hd, page, seed, spare_rows=0, q_size=1.5, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.n_head, self.n_kv, self.hd, self.page = lens, n_head, n_kv, hd, page
        need = [-(-(b + n) // page) for b, n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        rows = [n for _, n in lens]
        self.tokens = sum(rows)
        self.q_start = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
        self.kv_len = torch.tensor([b + n for b, n in lens], dtype=torch.int32)
        shape = (pages, n_kv, page, hd)
        self.codes = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in "kv"]
        self.scales = []
        for _ in "kv":
            s = torch.full(shape[:3], math.nan)
            for i, (b, n) in enumerate(lens):
                t = torch.arange(b + n)
                s[self.table[i].long()[t // page], :, t % page] = 0.02 * torch.exp(0.4 * torch.randn(b + n, n_kv, generator=g))
            self.scales.append(s)
        self.q = torch.randn(self.tokens + spare_rows, n_head * hd, generator=g) * q_size
        self.k = torch.randn(self.tokens + spare_rows, n_kv * hd, generator=g)
        self.v = torch.randn(self.tokens + spare_rows, n_kv * hd, generator=g)
        self.max_new, self.max_len = max(max(rows), 1), max(int(self.kv_len.max()), 1)
        for name in ("table", "kv_len", "q_start", "q", "k", "v"):
            setattr(self, name, getattr(self, name).to(device))
        self.codes, self.scales = [c.to(device) for c in self.codes], [s.to(device) for s in self.scales]

    def cache(self):
        return (*self.codes, *self.scales)


def attention(c, scale, absent=()):
    """(out, bound) [tokens][n_head * hd] in 64 bits.  ``absent``: (sequence, page index) pairs that the table lacks.

    The bound counts what the kernels round, each by its half step:
      the output to bf16: 2^-8 of the value;
      q and k to f16, or q to 15 bits of its largest: a score is off by at most
        d = scale * (2 * 2^-11 sum |q||k| + 2^-15 max|q| sum |k| + 2^-32 max(scale of k) sum |q|), the last for keys below f16's
        normal numbers; a weight by (e^(2d) - 1) of itself, numerator and sum alike;
      a weight, a value's scale and their product to f16: 3 * 2^-11 of |p v|, and below f16's normal numbers 2^-25 of the
        largest scale for each |code| and 2^-32 of the largest weight; or a weight times its value's scale to 15 bits of the
        largest of 32 neighbours: 2^-15 * 127 of that largest, for each of the 32;
      sums in 32 bits: 2^-20 of the sum of magnitudes, up to 16 additions deep after the matrix products."""
    hd, gqa = c.hd, c.n_head // c.n_kv
    out = torch.zeros(c.tokens, c.n_head * hd, dtype=torch.float64, device=c.q.device)
    bound = torch.zeros_like(out)
    row = 0
    for i, (before, new) in enumerate(c.lens):
        n = before + new
        if new == 0:
            continue
        t = torch.arange(n, device=c.q.device)
        keep = torch.ones(n, dtype=torch.bool, device=c.q.device)
        for s, p in absent:
            if s == i:
                keep &= t // c.page != p
        page, slot = c.table[i].long()[t // c.page].clamp_min(0), t % c.page
        seen = (t[None] <= torch.arange(before, n, device=c.q.device)[:, None]) & keep[None]
        for h in range(c.n_head):
            k = c.codes[0][page, h // gqa, slot].double() * torch.where(keep, c.scales[0][page, h // gqa, slot].double(), 0)[:, None]
            sv = torch.where(keep, c.scales[1][page, h // gqa, slot].double(), 0)
            v = c.codes[1][page, h // gqa, slot].double() * sv[:, None]
            q = c.q[row:row + new, h * hd:(h + 1) * hd].double()
            s = torch.where(seen, q @ k.T * scale, -math.inf)
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, 0, m))
            den = p.sum(1, keepdim=True)
            den = torch.where(den == 0, 1, den)
            o = p @ v / den
            d = scale * (2.0 ** -10 * q.abs() @ k.abs().T + 2.0 ** -15 * q.abs().amax(1, keepdim=True) * k.abs().sum(1)[None]
                         + 2.0 ** -32 * k.abs().amax() * q.abs().sum(1, keepdim=True))
            d = torch.where(seen, d, 0).amax(1, keepdim=True)
            size = p @ v.abs() / den
            top = torch.nn.functional.pad(p * sv, (0, -n % 32)).view(new, -(-n // 32), 32).amax(2).sum(1, keepdim=True) / den
            floor = 2.0 ** -25 * 127 * sv.abs().amax() + 2.0 ** -32 * v.abs().sum(0)[None] / den
            err = size * (torch.expm1(2 * d) + 3 * 2.0 ** -11 + 2.0 ** -20) + 32 * 2.0 ** -15 * 127 * top + floor
            out[row:row + new, h * hd:(h + 1) * hd] = o
            bound[row:row + new, h * hd:(h + 1) * hd] = 2.0 ** -8 * (o.abs() + err) + err
        row += new
    return out, bound


def store(c, theta):
    """Rotated q, and the four arrays after the store, in 64 bits (codes int8)."""
    hd, dev = c.hd, c.q.device
    pos = torch.cat([torch.arange(b, b + n, device=dev) for b, n in c.lens]).double()
    freq = theta ** (-2 * torch.arange(hd // 2, device=dev, dtype=torch.float64) / hd)
    cos, sin = torch.cos(pos[:, None] * freq)[:, None], torch.sin(pos[:, None] * freq)[:, None]

    def rotate(x):
        x = x[:c.tokens].double().view(c.tokens, -1, hd)
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    codes, scales = [x.clone() for x in c.codes], [x.clone() for x in c.scales]
    row = 0
    new = [rotate(c.k), c.v[:c.tokens].double().view(c.tokens, -1, hd)]
    for i, (before, n) in enumerate(c.lens):
        t = torch.arange(before, before + n, device=dev)
        page, slot = c.table[i].long()[t // c.page], t % c.page
        for j in (0, 1):
            x = new[j][row:row + n]
            top = x.abs().amax(-1)
            codes[j][page, :, slot] = (x * (torch.where(top > 0, top, 1).reciprocal() * 127)[..., None]).round().to(torch.int8)
            scales[j][page, :, slot] = (top / 127).float()
        row += n
    return rotate(c.q).view(c.tokens, -1), codes, scales
