"""Calls of the paged cache and its decoder that fail half way leave both as they were: lengths, pages and the device's arrays (on the
CPU, with a stand-in for the engine)."""
import contextlib

import pytest
import torch


class Lib:
    def s12_moe_gather_async(self, *args):
        return 0


class Engine:
    """Does nothing, and raises ``error`` at call number ``fail_at`` of ``name``."""
    lib = Lib()

    def __init__(self):
        self.name, self.fail_at, self.error, self.calls = None, 0, None, 0

    def fail(self, name, at, error):
        self.name, self.fail_at, self.error, self.calls = name, at, error, 0

    def attention_paged_workspace(self, *args):
        return torch.zeros(16)

    def __getattr__(self, name):
        def call(*args, **kw):
            if name == self.name:
                self.calls += 1
                if self.calls == self.fail_at:
                    raise self.error
        return call


@pytest.fixture
def decoder(monkeypatch):
    from turbo_lossless_b200 import DecoderConfig, PagedDecoder, paged
    monkeypatch.setattr(paged, "_stream", lambda *_: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda *_: contextlib.nullcontext())
    cfg = DecoderConfig(n_embd=16, n_head=2, n_head_kv=1, n_ff=8, n_vocab=10, n_layer=3, max_seq=64)
    layer = {k: None for k in ("wq", "wk", "wv", "wo", "w_gate", "w_up", "w_down")}
    norms = {f"{n}.{i}": None for n in ("attn_norm", "ffn_norm") for i in range(3)}
    norms["output_norm"] = None
    return PagedDecoder(cfg, [layer] * 3, None, torch.zeros(10, 16, dtype=torch.int16), norms, max_tokens=40, max_seqs=4, num_pages=8,
                        page_size=16, eng=Engine())


def state(cache):
    return (cache.sequences(), {s: (cache.length(s), cache.pages(s)) for s in cache.sequences()}, cache.free_pages, sorted(cache._free),
            list(cache._users), cache.block_table.tolist(), cache.kv_len.tolist())


def kept(cache, error, call):
    before = state(cache)
    with pytest.raises(error):
        call()
    assert state(cache) == before


@pytest.mark.parametrize("bad", [2 ** 31, -2 ** 40, "x", None])
def test_tokens_that_are_no_int32(decoder, bad):
    c = decoder.cache
    kept(c, Exception, lambda: decoder.prefill([[1, bad]]))
    a, b = decoder.prefill([[1, 2], [3] * 16])
    kept(c, Exception, lambda: decoder.step([a, b], [1, bad]))
    kept(c, Exception, lambda: decoder.prefill([[1] * 15, [bad]], [a, b]))
    kept(c, Exception, lambda: decoder.prefill([[1], [bad]]))
    decoder.step([a, b], [1, 1])
    assert (c.length(a), c.length(b)) == (3, 17)


@pytest.mark.parametrize("name,at", [("embed_lookup", 1), ("rope_store_kv_paged", 2), ("attention_paged", 1), ("attention_paged", 3), ("argmax", 1)])
@pytest.mark.parametrize("error", [RuntimeError("out of memory"), KeyboardInterrupt(), "S12Error"])
def test_a_launch_that_fails(decoder, name, at, error):
    from turbo_lossless_b200 import S12Error
    error = S12Error("refused") if error == "S12Error" else error
    c, e = decoder.cache, decoder.eng
    a, b = decoder.prefill([[1, 2], [3] * 16])
    for call in (lambda: decoder.step([a, b], [1, 1]), lambda: decoder.prefill([[1] * 15, [2]], [a, b]), lambda: decoder.prefill([[1] * 20, [2]])):
        e.fail(name, at, error)
        kept(c, type(error), call)
    e.fail(None, 0, None)
    decoder.step([a, b], [1, 1])
    assert (c.length(a), c.length(b)) == (3, 17)


def test_sequences_that_are_not_there(decoder):
    (a,) = decoder.prefill([[1, 2]])
    kept(decoder.cache, KeyError, lambda: decoder.step([a, 3], [1, 1]))
    kept(decoder.cache, KeyError, lambda: decoder.cache.release(3))
    kept(decoder.cache, KeyError, lambda: decoder.cache.fork(3))


@pytest.mark.parametrize("error", [RuntimeError("a copy failed"), KeyboardInterrupt()])
def test_page_copies_that_fail(decoder, error):
    c, e = decoder.cache, decoder.eng
    a, b = decoder.prefill([[1, 2], [3] * 20])
    c.release(a)
    e.fail("copy_pages", 1, error)
    kept(c, type(error), lambda: c.fork(b))
    e.fail("copy_pages", 1, error)
    kept(c, type(error), c.compact)
    e.fail(None, 0, None)
    assert c.compact() == 1
    c.fork(b)


def test_uploads_that_fail(decoder, monkeypatch):
    """The device's arrays follow with the next call that gets through."""
    c = decoder.cache
    a, b = decoder.prefill([[1] * 17, [3] * 20])
    c.release(a)
    upload = type(c)._upload

    def once(self):
        monkeypatch.setattr(type(self), "_upload", upload)
        raise RuntimeError("a copy to the device failed")

    for call in (c.add, lambda: c.extend({b: 30}), lambda: c.fork(b), lambda: c.release(b), c.compact, lambda: decoder.step([b], [1])):
        monkeypatch.setattr(type(c), "_upload", once)
        kept(c, RuntimeError, call)
    monkeypatch.setattr(type(c), "_upload", lambda self: (_ for _ in ()).throw(RuntimeError("none gets through")))
    before = state(c)
    for call in (c.add, lambda: c.extend({b: 30}), lambda: c.fork(b), lambda: c.release(b), c.compact, lambda: decoder.step([b], [1])):
        with pytest.raises(RuntimeError):
            call()
        assert state(c) == before
    monkeypatch.setattr(type(c), "_upload", upload)
    c.add()
    c.extend({b: 1})
    assert c.kv_len[b] == 21


@pytest.mark.parametrize("n_embd,n_head,n_kv", [(18, 4, 2), (100, 3, 1)])
def test_heads_that_do_not_fill_the_embedding_are_refused(n_embd, n_head, n_kv):
    """The o projection would read columns that the attention does not write, as ``Decoder`` says, too."""
    from turbo_lossless_b200 import DecoderConfig, PagedDecoder
    cfg = DecoderConfig(n_embd=n_embd, n_head=n_head, n_head_kv=n_kv, n_ff=8, n_vocab=10, n_layer=1, max_seq=64)
    with pytest.raises(ValueError, match="n_embd"):
        PagedDecoder(cfg, [], None, torch.zeros(10, n_embd, dtype=torch.int16), {}, max_tokens=8, max_seqs=2, eng=Engine())
