"""The operators of the paged INT8 key-value cache: cases, inputs, their plain form, and what they must give.

  store    rotation of q and k of packed tokens, quantisation of k and v, and the store into the cache's pages
  prompt   causal attention of whole prompts, or of chunks behind a cached prefix, packed sequences, grouped heads
  decode   attention of one new token per sequence
  copy     pages copied over all layers: forking a sequence, compacting a pool

The cache holds int8 codes [page][kv head][position][head_dim] and one fp32 scale per (page, kv head, position); a
sequence's position t lies in page ``table[sequence][t // page_size]``, row ``t % page_size``.  A value is code * scale,
scale = absmax / 127.  The queries of a sequence are its last positions.  Rows are fp32, outputs of the attention bf16.
"""
import math
import random

import torch

own = False

THETA = 10000.0                            # base of the rotation's angles, as the decoder's default


def listed():
    return [
        # one token of one user behind 255 positions: the smallest call of a decode step
        dict(name="store_b1", kind="store", heads=32, kv_heads=8, head_dim=128, seqs=1, new=1, new_least=1, prefix=255, page=64),
        # a server's batch of prompts of different lengths, packed
        dict(name="store_prompts", kind="store", heads=32, kv_heads=8, head_dim=128, seqs=9, new=1501, new_least=60, prefix=0, page=64),
        # a short question
        dict(name="prompt_29", kind="prompt", heads=32, kv_heads=8, head_dim=128, seqs=1, new=29, new_least=29, prefix=0, page=64),
        # a batch of prompts of different lengths, packed
        dict(name="prompt_packed", kind="prompt", heads=32, kv_heads=8, head_dim=128, seqs=11, new=1900, new_least=41, prefix=0, page=64),
        # a chunk of a long conversation behind what is cached already, 64 query heads
        dict(name="prompt_chunk", kind="prompt", heads=64, kv_heads=8, head_dim=128, seqs=3, new=517, new_least=333, prefix=6000, page=64),
        # a long document
        dict(name="prompt_12000", kind="prompt", heads=32, kv_heads=8, head_dim=128, seqs=1, new=12000, new_least=12000, prefix=0, page=64),
        # interactive generation with 256 positions in the cache
        dict(name="decode_b1_256", kind="decode", heads=32, kv_heads=8, head_dim=128, seqs=1, longest=256, least=256, page=64),
        # a mid-size batch of long contexts
        dict(name="decode_b24_4k", kind="decode", heads=32, kv_heads=8, head_dim=128, seqs=24, longest=4096, least=1900, page=64),
        # throughput serving: many sequences, short contexts, small pages
        dict(name="decode_b256_200", kind="decode", heads=32, kv_heads=8, head_dim=128, seqs=256, longest=320, least=70, page=16),
        # one GPU of eight that share a model with 8 kv heads: one kv head, a long context
        dict(name="decode_b2_65521", kind="decode", heads=8, kv_heads=1, head_dim=128, seqs=2, longest=65521, least=65521, page=128),
        # a fork: the last, partly filled page of one sequence
        dict(name="copy_1_page", kind="copy", kv_heads=8, head_dim=128, layers=32, pages=80, moves=1, page=64),
        # compacting a pool after many sequences ended
        dict(name="copy_300_pages", kind="copy", kv_heads=8, head_dim=128, layers=16, pages=777, moves=300, page=64),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (64, 8, 128), (8, 1, 128), (32, 32, 128), (16, 2, 64), (24, 8, 96), (4, 2, 64)])
    page = rng.choice([16, 32, 64, 128])
    kind = rng.choice(["store", "prompt", "prompt", "decode", "decode", "copy"])
    shape = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page)
    if kind in ("store", "prompt"):
        seqs = _log(rng, 1, 16)
        new = _log(rng, 1, 6000 // seqs)
        prefix = rng.choice([0, 0, _log(rng, 1, 7000)])
        return dict(kind=kind, seqs=seqs, new=new, new_least=rng.randint(max(1, new // 20), new), prefix=prefix, **shape)
    if kind == "decode":
        seqs = _log(rng, 1, 300)
        longest = _log(rng, 1, min(100000, 400000 // seqs))
        return dict(kind=kind, seqs=seqs, longest=longest, least=rng.randint(max(1, longest // 8), longest), **shape)
    pages = _log(rng, 40, 800)
    return dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, page=page, layers=_log(rng, 1, 16), pages=pages,
                moves=_log(rng, 1, pages * 2 // 5))


def _lengths(case):
    """[(cached before, new tokens)] of the sequences: the ends of the range first, then spread between them."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] == "decode":
        n = [case["longest"], case["least"]] + [r.randint(case["least"], case["longest"]) for _ in range(case["seqs"])]
        return [(x - 1, 1) for x in n[:case["seqs"]]]
    new = [case["new"], case["new_least"]] + [r.randint(case["new_least"], case["new"]) for _ in range(case["seqs"])]
    return [(r.randint(case["prefix"] // 2, case["prefix"]), x) for x in new[:case["seqs"]]]


def work(case):
    hd, hkv = case["head_dim"], case["kv_heads"]
    entry = hkv * (2 * hd + 8)                                        # bytes of a position: codes and scales
    if case["kind"] == "copy":
        return {"bytes": 2 * case["moves"] * case["layers"] * case["page"] * entry, "flops": 0}
    lens = _lengths(case)
    tokens, h = sum(n for _, n in lens), case["heads"]
    if case["kind"] == "store":
        return {"bytes": tokens * (4 * hd * (2 * h + 2 * hkv) + entry), "flops": tokens * hd * (3 * h + 5 * hkv)}
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in lens)
    return {"bytes": sum(p + n for p, n in lens) * entry + tokens * h * hd * 6, "flops": 4 * hd * h * pairs}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hd, hkv, ps = case["head_dim"], case["kv_heads"], case["page"]
    layers = case.get("layers", 1)
    if case["kind"] == "copy":
        pages, lens = case["pages"], []
    else:
        lens = _lengths(case)
        need = [-(-(p + n) // ps) for p, n in lens]
        pages = sum(need) + 3
    # codes as rows of normal values give them, scales of rows whose sizes differ
    shape = (layers, pages, hkv, ps, hd)
    s = dict(case=case, lens=lens)
    for x in "kv":
        codes = torch.empty(shape, device="cuda", dtype=torch.int8)
        for layer in range(layers):
            codes[layer] = (torch.randn(shape[1:], generator=g, device="cuda") * 45).round_().clamp_(-127, 127).to(torch.int8)
        s["codes_" + x] = codes
        s["scale_" + x] = torch.exp(0.3 * torch.randn(shape[:4], generator=g, device="cuda")) * (1 / 45)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    if case["kind"] == "copy":
        s["src"], s["dst"] = order[:case["moves"]].clone(), order[case["moves"]:2 * case["moves"]].clone()
        return s
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    h, tokens = case["heads"], sum(n for _, n in lens)
    s["table"] = table
    s["kv_len"] = torch.tensor([p + n for p, n in lens], dtype=torch.int32, device="cuda")
    s["q_start"] = torch.tensor([sum(n for _, n in lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    s["max_new"], s["max_len"] = max(n for _, n in lens), max(p + n for p, n in lens)
    s["q"] = torch.randn(tokens, h * hd, generator=g, device="cuda") * 1.5
    if case["kind"] == "store":
        s["k"] = torch.randn(tokens, hkv * hd, generator=g, device="cuda") * torch.exp(torch.randn(tokens, 1, generator=g, device="cuda") * 0.3)
        s["v"] = torch.randn(tokens, hkv * hd, generator=g, device="cuda")
        s["q_out"] = torch.empty_like(s["q"])
    else:
        s["out"] = torch.empty(tokens, h * hd, dtype=torch.int16, device="cuda")
    return s


_engines = {}


def _engine():
    if "e" not in _engines:
        from turbo_lossless_b200 import Split12Engine
        _engines["e"] = Split12Engine()
    return _engines["e"]


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c, e = s["case"], _engine()
    if c["kind"] == "copy":
        e.copy_pages(s["codes_k"], s["codes_v"], s["scale_k"], s["scale_v"], s["src"], s["dst"])
        return s["codes_k"], s["codes_v"], s["scale_k"], s["scale_v"]
    cache = s["codes_k"][0], s["codes_v"][0], s["scale_k"][0], s["scale_v"][0]
    if c["kind"] == "store":
        e.rope_store_kv_paged(s["q"], s["k"], s["v"], *cache, s["table"], s["kv_len"], s["q_start"], c["heads"], THETA, q_out=s["q_out"])
        return (s["q_out"], *cache)
    if "workspace" not in s:                                          # kept by the program, like the cache
        s["workspace"] = e.attention_paged_workspace(c["heads"], c["kv_heads"], c["head_dim"], len(s["lens"]), s["max_new"])
    e.attention_paged(s["q"], *cache, s["out"], s["table"], s["kv_len"], None if c["kind"] == "decode" else s["q_start"], c["heads"],
                      1 / math.sqrt(c["head_dim"]), s["max_new"], s["max_len"], workspace=s["workspace"])
    return s["out"].view(torch.bfloat16)


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "copy":
        for name in ("codes_k", "codes_v", "scale_k", "scale_v"):
            s[name][:, s["dst"]] = s[name][:, s["src"]]
        return s["codes_k"], s["codes_v"], s["scale_k"], s["scale_v"]
    if c["kind"] == "store":
        return _plain_store(s)
    return _plain_decode(s) if c["kind"] == "decode" else _plain_prompt(s)


def _plain_store(s):
    """In 64 bits: the angles of far positions, and codes next to a border."""
    c = s["case"]
    hd, ps = c["head_dim"], c["page"]
    tokens = s["q"].shape[0]
    row = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"], row, right=True) - 1
    pos = row - s["q_start"][seq + 1] + s["kv_len"][seq]
    freq = THETA ** (-2 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
    angle = (pos.double()[:, None] * freq)[:, None]
    cos, sin = angle.cos(), angle.sin()

    def rotate(x):
        lo, hi = x.double().view(tokens, -1, 2, hd // 2).unbind(2)
        return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], dim=2)

    page, slot = s["table"][seq, pos // ps].long(), (pos % ps).long()
    for name, x in (("k", rotate(s["k"])), ("v", s["v"].double().view(tokens, -1, hd))):
        top = x.abs().amax(2)
        s["codes_" + name][0][page, :, slot] = (x * (127 / top)[:, :, None]).round().clamp(-127, 127).nan_to_num(0).to(torch.int8)
        s["scale_" + name][0][page, :, slot] = (top / 127).float()
    s["q_out"] = rotate(s["q"]).view(tokens, -1).float()
    return s["q_out"], s["codes_k"][0], s["codes_v"][0], s["scale_k"][0], s["scale_v"][0]


def _plain_decode(s):
    """All sequences side by side, as long as the longest."""
    c = s["case"]
    h, hkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    seqs, pages = s["table"].shape
    table = s["table"].clamp_min(0).long()
    k, v = ((s["codes_" + x][0][table].float() * s["scale_" + x][0][table][..., None]).transpose(1, 2).reshape(seqs, hkv, -1, hd) for x in "kv")
    q = s["q"].view(seqs, hkv, h // hkv, hd) * (1 / math.sqrt(hd))
    absent = torch.arange(pages * c["page"], device="cuda") >= s["kv_len"][:, None]
    w = (q @ k.transpose(2, 3)).masked_fill_(absent[:, None, None], -math.inf)
    w = w.sub_(w.amax(3, keepdim=True)).exp_()
    return ((w @ v) / w.sum(3, keepdim=True)).view(seqs, h * hd).to(torch.bfloat16)


def _plain_prompt(s):
    c = s["case"]
    h, hkv, hd, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    got = []
    at = 0
    for i, (before, new) in enumerate(s["lens"]):
        n = before + new
        pages = s["table"][i, :-(-n // ps)].long()
        k, v = ((s["codes_" + x][0][pages].float() * s["scale_" + x][0][pages][..., None]).transpose(0, 1).reshape(hkv, 1, -1, hd)[:, :, :n]
                for x in "kv")
        q = s["q"][at:at + new].view(new, hkv, h // hkv, hd).permute(1, 2, 0, 3) * (1 / math.sqrt(hd))
        allowed = torch.arange(n, device="cuda") <= torch.arange(before, n, device="cuda")[:, None]
        out = []
        some = max(1, (1 << 29) // (new * n * h // hkv))                  # kv heads at a time: the scores are large
        for j in range(0, hkv, some):
            heads = slice(j, j + some)
            w = (q[heads] @ k[heads].transpose(2, 3)).masked_fill_(~allowed, -math.inf)
            w = w.sub_(w.amax(3, keepdim=True)).exp_()
            out.append((w @ v[heads]) / w.sum(3, keepdim=True))
        got.append(torch.cat(out).permute(2, 0, 1, 3).reshape(new, h * hd))
        at += new
    return torch.cat(got).to(torch.bfloat16)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        return None, None, *(s[x].double().index_copy(1, s["dst"].long(), s[x].double().index_select(1, s["src"].long()))
                             for x in ("scale_k", "scale_v"))
    hd, h, hkv, ps = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    if case["kind"] == "store":
        rows = []
        for before, new in s["lens"]:
            rows += range(before, before + new)
        pos = torch.tensor(rows, device="cuda", dtype=torch.float64)
        z = torch.view_as_complex(torch.stack(s["q"].double().view(len(rows), h, 2, hd // 2).unbind(2), -1))
        inv = torch.exp(torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) * (-math.log(THETA) / hd))
        turn = torch.polar(torch.ones_like(inv).expand(len(rows), -1), pos[:, None] * inv)
        z = z * turn[:, None]
        q = torch.cat([z.real, z.imag], -1).reshape(len(rows), h * hd)
        scale_k, scale_v = s["scale_k"][0].double(), s["scale_v"][0].double()
        zk = torch.view_as_complex(torch.stack(s["k"].double().view(len(rows), hkv, 2, hd // 2).unbind(2), -1)) * turn[:, None]
        top_k = torch.maximum(zk.real.abs(), zk.imag.abs()).amax(-1) / 127
        top_v = s["v"].double().view(len(rows), hkv, hd).abs().amax(-1) / 127
        r = 0
        for i, (before, new) in enumerate(s["lens"]):
            where = torch.arange(before, before + new, device="cuda")
            page, slot = s["table"][i].long()[where // ps], where % ps
            scale_k[page, :, slot] = top_k[r:r + new]
            scale_v[page, :, slot] = top_v[r:r + new]
            r += new
        return q, None, None, scale_k, scale_v
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    r = 0
    for i, (before, new) in enumerate(s["lens"]):
        where = torch.arange(before + new, device="cuda")
        page, slot = s["table"][i].long()[where // ps], where % ps
        seen = torch.tril(torch.ones(new, before + new, dtype=torch.bool, device="cuda"), diagonal=before)
        for head in range(h):
            kv = head * hkv // h
            k = s["codes_k"][0][page, kv, slot].double() * s["scale_k"][0][page, kv, slot].double()[:, None]
            v = s["codes_v"][0][page, kv, slot].double() * s["scale_v"][0][page, kv, slot].double()[:, None]
            x = s["q"][r:r + new, head * hd:(head + 1) * hd].double() @ k.T / math.sqrt(hd)
            out[r:r + new, head * hd:(head + 1) * hd] = torch.softmax(torch.where(seen, x, -math.inf), 1) @ v
        r += new
    return out
