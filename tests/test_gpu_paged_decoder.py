"""Prompts through ``PagedDecoder`` and on, against ``Decoder`` that takes the same tokens one at a time, and every call of the
paged operators on the way against 64 bits.

The two decoders round the same values to bf16 and int8, with sums in other orders: now and then a rounding falls the other
way, and the model carries it on.  How far is the model's own doing: the test moves every element of the embedding by up to
one step of bf16 (twice the half step that a rounding is off by), runs the token-by-token decoder again, and takes the largest
change of its logits as what roundings do to this model and text.  The decoders may differ by that and by 2 % of the largest
logit, which the decoder's own test against numpy allows each.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def model(seed=5, n_embd=256, n_head=4, n_head_kv=2):
    import torch
    from oracle import oracle as O, step_oracle as S
    from turbo_lossless_b200 import CompressedWeight, DecoderConfig
    cfg = DecoderConfig(n_embd=n_embd, n_head=n_head, n_head_kv=n_head_kv, n_ff=512, n_vocab=1000, n_layer=2, max_seq=256)
    rng = np.random.default_rng(seed)
    kv = cfg.kv_dim
    shapes = {"wq": (n_embd, n_embd), "wk": (kv, n_embd), "wv": (kv, n_embd), "wo": (n_embd, n_embd), "w_gate": (512, n_embd),
              "w_up": (512, n_embd), "w_down": (n_embd, 512)}
    pack = lambda M, K, s: CompressedWeight.from_packed(O.pack(O.synth_weights(M, K, s, std=0.06, outlier_frac=1e-3)))  # noqa: E731
    layers = [{nm: pack(M, K, 100 * li + i) for i, (nm, (M, K)) in enumerate(shapes.items())} for li in range(cfg.n_layer)]
    embd = S.f32_to_bf16(rng.standard_normal((cfg.n_vocab, n_embd)).astype(np.float32)).reshape(cfg.n_vocab, n_embd)
    names = [f"attn_norm.{i}" for i in range(cfg.n_layer)] + [f"ffn_norm.{i}" for i in range(cfg.n_layer)] + ["output_norm"]
    norms = {nm: torch.from_numpy((1.0 + 0.1 * rng.standard_normal(n_embd)).astype(np.float32)).cuda() for nm in names}
    return cfg, layers, pack(cfg.n_vocab, n_embd, 999), torch.from_numpy(embd).cuda(), norms


def one_by_one(parts, tokens):
    """Logits after each of ``tokens`` from the contiguous decoder."""
    import torch
    from turbo_lossless_b200 import Decoder
    cfg, layers, head, embd, norms = parts
    dec, got = Decoder(cfg, layers, head, embd, norms, batch=1), []
    for t, token in enumerate(tokens):
        dec.tokens.fill_(int(token))
        dec.positions.fill_(t)
        dec.forward()
        got.append(dec.logits[0].clone())
    torch.cuda.synchronize()
    return got


def close(got, parts, tokens):
    import torch
    cfg, layers, head, embd, norms = parts
    want, moved = one_by_one(parts, tokens)[-1], 0.0
    for seed in range(6):
        g = torch.Generator(device="cuda").manual_seed(seed)
        other = embd + torch.randint(-1, 2, embd.shape, generator=g, device="cuda", dtype=torch.int16)
        moved = max(moved, float((one_by_one((cfg, layers, head, other, norms), tokens)[-1] - want).abs().max()))
    assert float((got - want).abs().max()) <= moved + 2e-2 * float(want.abs().max())


def watched():
    """An engine that checks every paged store and attention of a run against 64 bits, on the inputs that the call had."""
    import torch
    import paged_oracle as PO
    from turbo_lossless_b200 import Split12Engine

    class Watched(Split12Engine):
        calls = 0

        @staticmethod
        def case(q, k, v, cache, table, kv_len, q_start, n_head):
            c = PO.Case.__new__(PO.Case)
            c.tokens, c.n_head, c.n_kv, c.page, c.hd = q.shape[0], n_head, *cache[0].shape[1:]
            starts = list(range(c.tokens + 1)) if q_start is None else q_start.tolist()
            c.lens = [(n - (b - a), b - a) for a, b, n in zip(starts, starts[1:], kv_len.tolist())]
            c.q, c.k, c.v, c.table = q.clone(), k, v, table
            c.codes, c.scales = [x.clone() for x in cache[:2]], [x.clone() for x in cache[2:]]
            return c

        def rope_store_kv_paged(self, q, k, v, kv_k, kv_v, scale_k, scale_v, table, kv_len, q_start, n_head, theta, **kw):
            c = self.case(q, k, v, (kv_k, kv_v, scale_k, scale_v), table, kv_len, q_start, n_head)
            super().rope_store_kv_paged(q, k, v, kv_k, kv_v, scale_k, scale_v, table, kv_len, q_start, n_head, theta, **kw)
            want, codes, scales = PO.store(c, theta)
            assert ((q.double() - want).abs() <= 5 * 2.0 ** -23 * c.q.abs().amax()).all()
            assert torch.equal(kv_k, codes[0]) and torch.equal(kv_v, codes[1])
            assert torch.equal(scale_k, scales[0]) and torch.equal(scale_v, scales[1])

        def attention_paged(self, q, kv_k, kv_v, scale_k, scale_v, out, table, kv_len, q_start, n_head, scale, *more):
            super().attention_paged(q, kv_k, kv_v, scale_k, scale_v, out, table, kv_len, q_start, n_head, scale, *more)
            c = self.case(q, None, None, (kv_k, kv_v, scale_k, scale_v), table, kv_len, q_start, n_head)
            want, bound = PO.attention(c, scale)
            assert ((out.view(torch.bfloat16).double() - want).abs() <= bound).all()
            Watched.calls += 1

    return Watched()


@pytest.mark.parametrize("heads,page", [((4, 2), 16), ((2, 1), 64), ((4, 4), 32)])
def test_prompts_steps_forks_and_compaction_match_the_token_by_token_decoder(heads, page):
    import torch
    from turbo_lossless_b200 import PagedDecoder
    parts = model(n_head=heads[0], n_head_kv=heads[1])
    rng = np.random.default_rng(1)
    text = [rng.integers(0, 1000, n).tolist() for n in (1, 40, 77, 130)]
    dec = PagedDecoder(*parts, max_tokens=300, max_seqs=6, page_size=page, eng=watched())
    seqs = dec.prefill(text)
    logits = dec.logits[:4].clone()
    for i in range(4):
        close(logits[i], parts, text[i])
        assert int(dec.next_tokens[i]) == int(logits[i].argmax())
    # a chunk behind what is cached, next to a single token
    more = [rng.integers(0, 1000, 20).tolist(), [3]]
    dec.prefill(more, [seqs[1], seqs[3]])
    text[1] += more[0]
    text[3] += more[1]
    logits = dec.logits[:2].clone()
    close(logits[0], parts, text[1])
    close(logits[1], parts, text[3])
    # a fork goes its own way; a sequence ends, the pool is compacted, the others go on
    twin = dec.cache.fork(seqs[1])
    dec.cache.release(seqs[2])
    assert dec.cache.compact() > 0
    batch = {seqs[0]: text[0], seqs[1]: text[1], twin: list(text[1]), seqs[3]: text[3]}
    for step in range(3):
        new = rng.integers(0, 1000, 4).tolist()
        for t, tokens in zip(new, batch.values()):
            tokens.append(t)
        logits = dec.step(list(batch), new)
    for i, tokens in enumerate(batch.values()):
        close(logits[i], parts, tokens)
    torch.cuda.synchronize()
    assert dec.eng.device_status() == 0 and dec.eng.calls == 2 * 5


def test_what_does_not_fit_leaves_the_decoder_as_it_was():
    from turbo_lossless_b200 import PagedCacheFull, PagedDecoder
    dec = PagedDecoder(*model(), max_tokens=50, max_seqs=2, num_pages=3, page_size=16)
    for prompts in ([[1] * 51], [[1], []], [[1], [1], [1]], [[1] * 49], []):
        with pytest.raises((ValueError, PagedCacheFull)):
            dec.prefill(prompts)
        assert dec.cache.sequences() == [] and dec.cache.free_pages == 3
    (a,) = dec.prefill([[1] * 40])
    with pytest.raises(ValueError):
        dec.step([a, a], [1, 1])
    with pytest.raises(PagedCacheFull):
        dec.prefill([[1] * 9], [a])
    assert dec.cache.length(a) == 40
