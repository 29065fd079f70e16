"""A prefill of more rows than one sequence tile of the projections' GEMM: every paged call against 64 bits, two prompts against the
token-by-token decoder."""
import pytest

from test_gpu_paged_decoder import close, model, watched

pytestmark = pytest.mark.gpu


def test_a_thousand_packed_rows():
    import numpy as np
    import torch
    from turbo_lossless_b200 import PagedDecoder
    parts = model(n_head=4, n_head_kv=2)
    rng = np.random.default_rng(2)
    text = [rng.integers(0, 1000, n).tolist() for n in (201, 7, 190, 222, 180, 64, 150)]
    dec = PagedDecoder(*parts, max_tokens=1100, max_seqs=8, page_size=32, eng=watched())
    seqs = dec.prefill(text)
    logits = dec.logits[:7].clone()
    for i in (0, 3):
        close(logits[i], parts, text[i])
    # a chunk and single tokens in one call
    more = [rng.integers(0, 1000, 30).tolist()] + [[int(t)] for t in rng.integers(0, 1000, 6)]
    dec.prefill(more, seqs)
    logits = dec.logits[:7].clone()
    for i in (0, 1):
        close(logits[i], parts, text[i] + more[i])
    torch.cuda.synchronize()
    assert dec.eng.device_status() == 0 and dec.eng.calls == 2 * 2
