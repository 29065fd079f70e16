"""A paged INT8 key-value cache and a decoder that runs whole prompts through it.

The reference engine keeps one contiguous cache and feeds a prompt token by token (engine/inference.cpp:198-366).
Here sequences of different lengths share one pool of pages: ``PagedKVCache`` hands pages out, forks a sequence by
sharing its full pages, frees and compacts; ``PagedDecoder`` runs packed prompts (or chunks of them) in one pass and
decodes all sequences side by side.  Device work is launches of the CUDA library; page bookkeeping is the host's.
"""
from __future__ import annotations

import contextlib
import heapq
from typing import Dict, List, Optional, Sequence

import torch

from .capi import check
from .decoder import DecoderConfig
from .engine import CompressedWeight, Split12Engine, _ptr, _stream


class PagedCacheFull(RuntimeError):
    """No page or sequence is free; the cache is as it was before the call."""


class PagedKVCache:
    """``n_layer`` layers of ``num_pages`` pages and the page lists of up to ``max_seqs`` sequences.

    ``kv_k`` / ``kv_v`` int8 [layer][page][kv head][position][head_dim], ``scale_k`` / ``scale_v`` fp32 without the last;
    ``block_table`` int32 [max_seqs][max_pages] and ``kv_len`` int32 [max_seqs] on the device follow the host's lists after
    every call, in place, so that a captured graph may read them.  Calls are ordered on the current stream.  A call that raises
    leaves everything as it was.
    """

    def __init__(self, n_layer: int, num_pages: int, n_head_kv: int, head_dim: int, page_size: int = 64, max_seqs: int = 8,
                 max_pages: Optional[int] = None, device="cuda", eng: Optional[Split12Engine] = None):
        if min(n_layer, num_pages, n_head_kv, head_dim, max_seqs) < 1 or page_size < 16 or page_size & (page_size - 1):
            raise ValueError("sizes must be positive, page_size a power of two from 16")
        self.page_size, self.num_pages, self.max_seqs = page_size, num_pages, max_seqs
        self.max_pages = num_pages if max_pages is None else max_pages
        self.eng = eng
        shape = (n_layer, num_pages, n_head_kv, page_size)
        self.kv_k = torch.zeros(*shape, head_dim, dtype=torch.int8, device=device)
        self.kv_v = torch.zeros_like(self.kv_k)
        self.scale_k = torch.zeros(shape, dtype=torch.float32, device=device)
        self.scale_v = torch.zeros_like(self.scale_k)
        self.block_table = torch.full((max_seqs, self.max_pages), -1, dtype=torch.int32, device=device)
        self.kv_len = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self._table = torch.full((max_seqs, self.max_pages), -1, dtype=torch.int32)
        self._free: List[int] = list(range(num_pages))                # a heap: the lowest page first
        self._users = [0] * num_pages                                 # sequences that hold the page
        self._pages: Dict[int, List[int]] = {}
        self._len: Dict[int, int] = {}

    # -- what is there ---------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> List[int]:
        return sorted(self._pages)

    def length(self, seq: int) -> int:
        return self._len[seq]

    def pages(self, seq: int) -> List[int]:
        return list(self._pages[seq])

    def layer(self, i: int):
        """The four arrays of one layer."""
        return self.kv_k[i], self.kv_v[i], self.scale_k[i], self.scale_v[i]

    # -- host bookkeeping ------------------------------------------------------
    def _take(self) -> int:
        page = heapq.heappop(self._free)
        self._users[page] = 1
        return page

    def _upload(self) -> None:
        self._table.fill_(-1)
        lens = [0] * self.max_seqs
        for seq, pages in self._pages.items():
            if pages:
                self._table[seq, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            lens[seq] = self._len[seq]
        self.block_table.copy_(self._table)                           # from pageable memory: read before the call returns
        self.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))

    def _follow(self) -> None:
        """After a failure: the device's arrays follow the lists, or do so with the next call that gets through."""
        with contextlib.suppress(Exception):
            self._upload()

    @contextlib.contextmanager
    def _or_as_before(self):
        """The lists go back to what they were when the block raises."""
        before = list(self._free), list(self._users), {seq: list(pages) for seq, pages in self._pages.items()}, dict(self._len)
        try:
            yield
        except BaseException:
            self._free, self._users, self._pages, self._len = before
            self._follow()
            raise

    def _shorten(self, lens: Dict[int, int]) -> None:
        """Sequences back to the lengths they had: the pages behind are free again.  As ``_or_as_before``, of these sequences alone."""
        for seq, n in lens.items():
            pages = self._pages[seq]
            while len(pages) > -(-n // self.page_size):
                self._drop(pages.pop())
            self._len[seq] = n
        self._follow()

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            heapq.heappush(self._free, page)

    def _copy(self, src: Sequence[int], dst: Sequence[int]) -> None:
        if not src:
            return
        both = torch.tensor([list(src), list(dst)], dtype=torch.int32).to(self.kv_k.device)
        self.eng = self.eng or Split12Engine()
        with torch.cuda.device(self.kv_k.device):
            self.eng.copy_pages(self.kv_k, self.kv_v, self.scale_k, self.scale_v, both[0], both[1])

    def _slot(self) -> int:
        for seq in range(self.max_seqs):
            if seq not in self._pages:
                return seq
        raise PagedCacheFull(f"all {self.max_seqs} sequences are in use")

    # -- sequences -------------------------------------------------------------
    def add(self) -> int:
        """A new, empty sequence: its row in ``block_table`` and ``kv_len``."""
        seq = self._slot()
        with self._or_as_before():
            self._pages[seq], self._len[seq] = [], 0
            self._upload()
        return seq

    def extend(self, new: Dict[int, int]) -> None:
        """Room for ``new[seq]`` more positions of each sequence, counted in ``kv_len``: all of them, or none."""
        need = {}
        for seq, n in new.items():
            if n < 0:
                raise ValueError(f"sequence {seq}: {n} new positions")
            pages = -(-(self._len[seq] + n) // self.page_size)
            if pages > self.max_pages:
                raise PagedCacheFull(f"sequence {seq} needs {pages} pages of {self.max_pages}")
            need[seq] = pages - len(self._pages[seq])
        if sum(need.values()) > len(self._free):
            raise PagedCacheFull(f"{sum(need.values())} pages needed, {len(self._free)} free")
        before = {seq: self._len[seq] for seq in new}
        try:
            for seq, n in new.items():
                for _ in range(need[seq]):
                    self._pages[seq].append(self._take())
                self._len[seq] += n
            self._upload()
        except BaseException:
            self._shorten(before)
            raise

    def fork(self, seq: int) -> int:
        """A new sequence with the same positions: full pages are shared (nobody writes them again), a last page with room
        is copied."""
        pages, n = self._pages[seq], self._len[seq]
        child = self._slot()
        full = n // self.page_size
        if len(pages) > full and not self._free:
            raise PagedCacheFull("a fork needs one free page")
        with self._or_as_before():
            mine = pages[:full]
            for page in mine:
                self._users[page] += 1
            if len(pages) > full:
                mine.append(self._take())
                self._copy([pages[full]], [mine[full]])
            self._pages[child], self._len[child] = mine, n
            self._upload()
        return child

    def release(self, seq: int) -> None:
        """Ends a sequence; pages that no other sequence holds are free again."""
        with self._or_as_before():
            for page in self._pages.pop(seq):
                self._drop(page)
            del self._len[seq]
            self._upload()

    def compact(self) -> int:
        """Moves pages so that those in use are the pool's first ones; returns how many were moved."""
        used = self.num_pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        moved = [p for p in range(used, self.num_pages) if self._users[p]]
        if not moved:
            return 0
        with self._or_as_before():
            self._copy(moved, holes)
            to = dict(zip(moved, holes))
            for a, b in to.items():
                self._users[b], self._users[a] = self._users[a], 0
            for pages in self._pages.values():
                pages[:] = [to.get(p, p) for p in pages]
            self._free = list(range(used, self.num_pages))
            self._upload()
        return len(moved)


class PagedDecoder:
    """A decoder (weights as for ``Decoder``) over a ``PagedKVCache``: ``prefill`` runs packed prompts or chunks in one
    pass, ``step`` one token of every given sequence.  ``max_tokens`` bounds the tokens of a call.  A call that raises leaves
    the sequences as they were."""

    def __init__(self, cfg: DecoderConfig, layers: List[Dict[str, CompressedWeight]], lm_head: CompressedWeight, token_embd: torch.Tensor,
                 norms: Dict[str, torch.Tensor], max_tokens: int, max_seqs: int = 8, num_pages: Optional[int] = None, page_size: int = 64,
                 eng: Optional[Split12Engine] = None):
        self.cfg, self.layers, self.lm_head, self.token_embd, self.norms = cfg, layers, lm_head, token_embd, norms
        if cfg.n_head * cfg.head_dim != cfg.n_embd:
            raise ValueError(f"the attention output feeds the o projection: {cfg.n_head} heads of {cfg.head_dim} are not n_embd {cfg.n_embd}")
        self.eng = eng or Split12Engine()
        self.max_tokens = max(max_tokens, max_seqs)
        dev, n, hd, T = token_embd.device, cfg.n_embd, cfg.head_dim, self.max_tokens
        max_pages = -(-cfg.max_seq // page_size)
        self.cache = PagedKVCache(cfg.n_layer, max_seqs * max_pages if num_pages is None else num_pages, cfg.n_head_kv, hd, page_size,
                                  max_seqs, max_pages, dev, self.eng)
        f32, i32 = dict(device=dev, dtype=torch.float32), dict(device=dev, dtype=torch.int32)
        self.hidden, self.hidden2 = torch.zeros(T, n, **f32), torch.zeros(T, n, **f32)
        self.q_buf = torch.zeros(T, cfg.n_head * hd, **f32)
        self.k_buf, self.v_buf = torch.zeros(T, cfg.kv_dim, **f32), torch.zeros(T, cfg.kv_dim, **f32)
        self.ffn_gate, self.ffn_up = torch.zeros(T, cfg.n_ff, **f32), torch.zeros(T, cfg.n_ff, **f32)
        self.bf16_a = torch.zeros(T, n, device=dev, dtype=torch.int16)
        self.bf16_b = torch.zeros(T, cfg.n_ff, device=dev, dtype=torch.int16)
        self.last = torch.zeros(max_seqs, n, device=dev, dtype=torch.int16)
        self.logits = torch.zeros(max_seqs, cfg.n_vocab, **f32)
        self.next_tokens = torch.zeros(max_seqs, **i32)
        self.workspace = self.eng.attention_paged_workspace(cfg.n_head, cfg.n_head_kv, hd, max_seqs, self.max_tokens, dev)

    def _proj(self, ws, x, outs, rows: int) -> None:
        e = self.eng
        if rows == 1:
            e.gemv(ws, x, outs)
        elif rows <= 16:
            for w, o in zip(ws, outs):
                e.gemv_batched(w, x, o, x.stride(0), o.stride(0), rows)
        else:
            e.gemm_multi(ws, x, outs, x.stride(0), rows)

    def _forward(self, seqs: List[int], tokens: List[List[int]]) -> torch.Tensor:
        """Logits [len(seqs)][vocabulary] after the last of each sequence's new tokens (the decoder's own buffer)."""
        new = [len(t) for t in tokens]
        rows, S = sum(new), len(seqs)
        if len(new) != S or len(set(seqs)) != S or S == 0 or min(new) < 1 or rows > self.max_tokens:
            raise ValueError(f"needs distinct sequences with at least a token each, {self.max_tokens} tokens at most")
        dev, before = self.token_embd.device, {s: self.cache.length(s) for s in seqs}
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        # what the host knows of this call, in one copy
        host = torch.tensor([t for ts in tokens for t in ts] + starts + [s - 1 for s in starts[1:]] + [S] + list(seqs), dtype=torch.int32)
        meta = host.to(dev)
        self.cache.extend(dict(zip(seqs, new)))
        try:
            return self._run(seqs, new, meta)
        except BaseException:
            self.cache._shorten(before)
            raise

    def _run(self, seqs: List[int], new: List[int], meta: torch.Tensor) -> torch.Tensor:
        c, e, rows, S = self.cfg, self.eng, sum(new), len(seqs)
        hd, scale = c.head_dim, 1.0 / float(c.head_dim) ** 0.5
        ids, q_start, ends, count = meta[:rows], meta[rows:rows + S + 1], meta[rows + S + 1:rows + 2 * S + 1], meta[rows + 2 * S + 1:rows + 2 * S + 2]
        order = meta[rows + 2 * S + 2:].long()
        table, kv_len = self.cache.block_table[order], self.cache.kv_len[order]
        q_start = None if rows == S else q_start
        max_new, max_len = max(new), max(self.cache.length(s) for s in seqs)
        cur, res = self.hidden[:rows], self.hidden2[:rows]
        q, k, v, gate, up = self.q_buf[:rows], self.k_buf[:rows], self.v_buf[:rows], self.ffn_gate[:rows], self.ffn_up[:rows]
        a, b = self.bf16_a[:rows], self.bf16_b[:rows]
        e.embed_lookup(self.token_embd, ids, cur)
        e.rms_norm_bf16(cur, self.norms["attn_norm.0"], a, c.rms_norm_eps, rows)
        for li, L in enumerate(self.layers):
            kv = self.cache.layer(li)
            self._proj([L["wq"], L["wk"], L["wv"]], a, [q, k, v], rows)
            e.rope_store_kv_paged(q, k, v, *kv, table, kv_len, q_start, c.n_head, c.rope_theta)
            e.attention_paged(q, *kv, a, table, kv_len, q_start, c.n_head, scale, max_new, max_len, self.workspace)
            self._proj([L["wo"]], a, [res], rows)
            e.rms_norm_bf16(res, self.norms[f"ffn_norm.{li}"], a, c.rms_norm_eps, rows, residual=cur)
            self._proj([L["w_gate"], L["w_up"]], a, [gate, up], rows)
            e.silu_mul_bf16(gate, up, b, c.n_ff, rows)
            self._proj([L["w_down"]], b, [cur], rows)
            nxt = self.norms[f"attn_norm.{li + 1}"] if li + 1 < len(self.layers) else self.norms["output_norm"]
            e.rms_norm_bf16(cur, nxt, a, c.rms_norm_eps, rows, residual=res)
        last = a
        if rows != S:                                                  # the rows that are a sequence's last token
            last = self.last[:S]
            check(e.lib.s12_moe_gather_async(_ptr(a), c.n_embd, S, 1, S, _ptr(ends), _ptr(count), _ptr(last), _stream()), "s12_moe_gather_async")
        logits = self.logits[:S]
        self._proj([self.lm_head], last, [logits], S)
        e.argmax(logits, self.next_tokens[:S])
        return logits

    def prefill(self, prompts: Sequence[Sequence[int]], seqs: Optional[Sequence[int]] = None) -> List[int]:
        """Runs the prompts through the model in one pass and returns their sequences: new ones, or, with ``seqs``, the given
        ones go on (the next chunk of a long prompt).  ``logits[i]`` / ``next_tokens[i]`` then belong to prompt i."""
        seqs = list(seqs) if seqs is not None else None
        if seqs is None:
            with self.cache._or_as_before():
                made = [self.cache.add() for _ in prompts]
                self._forward(made, [list(p) for p in prompts])
            return made
        self._forward(seqs, [list(p) for p in prompts])
        return seqs

    def step(self, seqs: Sequence[int], tokens: Sequence[int]) -> torch.Tensor:
        """One token of every given sequence; returns the logits [len(seqs)][vocabulary]."""
        return self._forward(list(seqs), [[int(t)] for t in tokens])
