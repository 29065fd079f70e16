"""The paged cache on the CPU: its bookkeeping, and what the entry points refuse before any device work."""
import ctypes as C
import random

import pytest
import torch


class FakeEngine:
    """Copies pages as the device would, without one."""

    def copy_pages(self, kv_k, kv_v, scale_k, scale_v, src, dst):
        src, dst = src.long(), dst.long()
        assert len(set(dst.tolist())) == len(dst) and not set(dst.tolist()) & set(src.tolist())
        for x in (kv_k, kv_v, scale_k, scale_v):
            x[:, dst] = x[:, src]


@pytest.fixture
def cache(monkeypatch):
    from turbo_lossless_b200 import PagedKVCache
    c = PagedKVCache(2, 24, 2, 4, page_size=16, max_seqs=5, max_pages=8, device="cpu", eng=FakeEngine())
    import contextlib
    monkeypatch.setattr(torch.cuda, "device", lambda *_: contextlib.nullcontext())
    return c


def value(seq_id, t):
    return float(seq_id * 1000 + t)


def write(c, seq, ident, lo, hi):
    for t in range(lo, hi):
        c.scale_k[:, c.pages(seq)[t // 16], :, t % 16] = value(ident, t)


def read(c, seq):
    return [c.scale_k[1, int(c.block_table[seq, t // 16]), 1, t % 16].item() for t in range(int(c.kv_len[seq]))]


def test_sequences_keep_their_positions_through_forks_releases_and_compaction(cache):
    """Random use against lists: every sequence reads back what was written for it, pages are counted right."""
    from turbo_lossless_b200 import PagedCacheFull
    c, rng, want, fresh = cache, random.Random(3), {}, iter(range(10**6))
    for step in range(600):
        what = rng.choice(["add", "extend", "extend", "extend", "fork", "release", "compact"])
        try:
            if what == "add":
                s = c.add()
                want[s] = []
            elif what == "extend" and want:
                chosen = rng.sample(sorted(want), rng.randint(1, len(want)))
                new = {s: rng.choice([0, 1, 1, 5, 16, 33]) for s in chosen}
                before = (c.free_pages, {s: c.length(s) for s in want})
                try:
                    c.extend(new)
                except PagedCacheFull:
                    assert before == (c.free_pages, {s: c.length(s) for s in want})
                    raise
                for s, n in new.items():
                    ident, lo = next(fresh), len(want[s])
                    write(c, s, ident, lo, lo + n)
                    want[s] = want[s] + [value(ident, t) for t in range(lo, lo + n)]
            elif what == "fork" and want:
                s = rng.choice(sorted(want))
                want[c.fork(s)] = list(want[s])
            elif what == "release" and want:
                s = rng.choice(sorted(want))
                c.release(s)
                del want[s]
            elif what == "compact":
                c.compact()
                used = {p for s in want for p in c.pages(s)}
                assert used == set(range(len(used)))
                assert c.compact() == 0
        except PagedCacheFull:
            pass
        used = {p for s in want for p in c.pages(s)}
        assert c.free_pages == c.num_pages - len(used) and c.sequences() == sorted(want)
        for s, values in want.items():
            assert read(c, s) == values and len(c.pages(s)) == -(-len(values) // 16)
            assert c.block_table[s, len(c.pages(s)):].eq(-1).all()
        for s in range(c.max_seqs):
            assert s in want or (int(c.kv_len[s]) == 0 and c.block_table[s].eq(-1).all())


def test_a_full_cache_and_wrong_sizes_are_refused(cache):
    from turbo_lossless_b200 import PagedCacheFull, PagedKVCache
    a, b = cache.add(), cache.add()
    with pytest.raises(PagedCacheFull):
        cache.extend({a: 129})                                        # nine pages of eight
    cache.extend({a: 128, b: 128})
    d = cache.fork(a)                                                 # full pages only: no page is taken
    assert cache.free_pages == 8
    e = cache.add()
    cache.extend({e: 113})
    with pytest.raises(PagedCacheFull):
        cache.fork(e)                                                 # its last page has room: one page would be needed
    with pytest.raises(ValueError):
        cache.extend({e: -1})
    cache.release(a)
    assert cache.free_pages == 0                                      # the fork still holds them
    cache.release(d)
    assert cache.free_pages == 8
    for _ in range(3):
        cache.add()
    with pytest.raises(PagedCacheFull):
        cache.add()
    with pytest.raises(KeyError):
        cache.extend({9: 1})
    for bad in (dict(page_size=24), dict(page_size=8), dict(n_layer=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_layer=1, num_pages=4, n_head_kv=1, head_dim=4, device="cpu"), **bad})


def good():
    from turbo_lossless_b200.capi import S12PagedBatch, S12PagedKv
    p = 4096
    return S12PagedKv(p, p, p, p, 10, 16, 2, 128), S12PagedBatch(p, p, p, 3, 4, 4, 7, 3, 50)


KV_EDITS = [dict(k=None), dict(v=None), dict(scale_k=None), dict(scale_v=None), dict(k=4097), dict(scale_v=4100), dict(num_pages=0), dict(page_size=8),
            dict(page_size=48), dict(page_size=2048), dict(n_head_kv=0), dict(head_dim=0), dict(head_dim=126), dict(head_dim=260)]
BATCH_EDITS = [dict(block_table=None), dict(kv_len=None), dict(num_seqs=0), dict(num_tokens=0), dict(table_pages=0), dict(table_stride=3), dict(q_start=None)]


def test_entry_points_refuse_before_any_device_work():
    """Every refusal is a negative code with a text that names the call; no device is needed for it."""
    from turbo_lossless_b200 import capi
    lib, p = capi.load(), 4096
    store = lambda kv, b, q=p, qs=512, k=p, v=p, ks=256, o=p, os=512, h=4, th=1e4: lib.s12_rope_store_kv_paged_async(  # noqa: E731
        q, qs, k, v, ks, o, os, C.byref(kv) if kv else None, C.byref(b) if b else None, h, th, None)
    attend = lambda kv, b, q=p, qs=512, o=p, os=512, h=4, ws=p, n=1 << 40, sc=0.1: lib.s12_attention_paged_async(  # noqa: E731
        q, qs, C.byref(kv) if kv else None, C.byref(b) if b else None, o, os, h, sc, ws, n, None)
    copy = lambda kv, layers=2, s=p, d=p, n=1: lib.s12_copy_pages_async(C.byref(kv) if kv else None, layers, s, d, n, None)  # noqa: E731

    def refused(rc, name):
        assert rc < 0 and rc != -3, rc                                # not an error of CUDA
        assert name in lib.s12_last_error()

    for edit in KV_EDITS:
        kv, b = good()
        for f, x in edit.items():
            setattr(kv, f, x)
        refused(store(kv, b), b"s12_rope_store_kv_paged_async")
        refused(attend(kv, b), b"s12_attention_paged_async")
        refused(copy(kv), b"s12_copy_pages_async")
    for edit in BATCH_EDITS:
        kv, b = good()
        for f, x in edit.items():
            setattr(b, f, x)
        refused(store(kv, b), b"s12_rope_store_kv_paged_async")
        refused(attend(kv, b), b"s12_attention_paged_async")
    kv, b = good()
    for edit in (dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(qs=511), dict(os=511), dict(ks=255), dict(h=3), dict(h=1), dict(h=0),
                 dict(th=0.0), dict(th=-1.0), dict(th=float("nan")), dict(th=float("inf"))):
        refused(store(kv, b, **edit), b"s12_rope_store_kv_paged_async")
    for edit in (dict(q=None), dict(o=None), dict(qs=511), dict(os=511), dict(h=3), dict(h=0), dict(sc=float("nan")), dict(sc=float("inf"))):
        refused(attend(kv, b, **edit), b"s12_attention_paged_async")
    for f in ("max_new", "max_len"):
        kv, b = good()
        setattr(b, f, 0)
        refused(attend(kv, b), b"s12_attention_paged_async")
    kv, b = good()
    refused(store(None, b), b"s12_rope_store_kv_paged_async")
    refused(attend(kv, None), b"s12_attention_paged_async")
    refused(copy(None), b"s12_copy_pages_async")
    for edit in (dict(layers=0), dict(layers=70000), dict(s=None), dict(d=None), dict(n=-1)):
        refused(copy(kv, **edit), b"s12_copy_pages_async")
    large, _ = good()
    large.page_size = 1024
    refused(copy(large, n=1 << 30), b"s12_copy_pages_async")          # more blocks than a grid has
    assert copy(kv, n=0) == 0 and copy(kv, s=None, d=None, n=0) == 0
    for sizes in ((0, 1, 128, 1, 1), (8, 0, 128, 1, 1), (8, 1, 0, 1, 1), (8, 1, 128, 0, 1), (8, 1, 128, 1, 0)):
        refused(lib.s12_attention_paged_workspace_bytes(*sizes), b"s12_attention_paged_workspace_bytes")


def test_structs_match_the_header():
    from turbo_lossless_b200.capi import S12PagedBatch, S12PagedKv
    assert C.sizeof(S12PagedKv) == 4 * 8 + 4 * 4 and C.sizeof(S12PagedBatch) == 3 * 8 + 6 * 4
