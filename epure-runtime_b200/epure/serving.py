"""Several sequences decoding together through a ``PackedDecoder``'s weights over a paged key-value cache.

The reference decodes through the Hugging Face model around its packed linears, one dense cache a sequence.
``PackedDecoder`` (epure.model) runs one sequence over a static cache.  ``BatchDecoder`` runs the same block for a
batch: the packed linears take the batch as rows, and per layer one launch normalises (Qwen3) and rotates q and k
and writes k and v into the cache's pages, quantised where the cache is 8-bit (``epure.paged.write``), and one
attends over every sequence's pages (``epure.paged.attend``).  A prompt's rows go through the same write; its
attention reads the sequence's rows back (``epure.paged.read``) and runs torch's SDPA on them, so it sees what the
steps after it will see.

    decoder = PackedDecoder(shapes, max_len=4096)
    batch = BatchDecoder(decoder, seqs=16, format="int8")
    tokens = batch.generate(prompts, n_new=64)        # greedy, one CUDA graph a step
    tokens = batch.generate(prompts, n_new=64, prefix=system)       # behind a prompt that all have in common
    tokens, passes = batch.speculate(prompts, n_new=64, drafts=4)   # drafted tokens, judged several at a time

With ``sparse`` a step attends over the blocks that ``epure.paged.select`` chooses, not over the whole cache.
"""
import math

import torch
import torch.nn.functional as F

from . import _native, paged, sampling


class BatchDecoder:
    """``decoder``: a ``PackedDecoder`` in mode "ours" (its stores, embedding, lm_head and rotary tables are used, its
    own cache is not).  ``seqs`` sequences of up to the decoder's ``max_len`` tokens; ``pages`` defaults to room for
    all of them.  ``format``: "same", "int8" or "fp8".  ``sparse``: (count, sinks, recent) blocks of ``page_size`` tokens
    that each step's attention reads, as ``paged.select`` takes them; None: all."""

    def __init__(self, decoder, seqs=16, format="same", page_size=64, pages=None, sparse=None):
        if decoder.mode != "ours" or decoder.dtype != torch.bfloat16:
            raise ValueError("epure: a BatchDecoder needs a PackedDecoder in linear_mode 'ours'")
        sh = decoder.shapes
        self.decoder, self.shapes, self.device = decoder, sh, decoder.device
        per_seq = -(-decoder.max_len // page_size)
        self.cache = paged.PagedKVCache(decoder.layers, pages or seqs * per_seq, page_size, sh.kv_heads, sh.head_dim,
                                        seqs, decoder.max_len, format, decoder.dtype, decoder.device,
                                        bounds=sparse is not None)
        if sparse is not None:
            count, sinks, recent = sparse
            if min(sinks, recent) < 0 or count < max(1, sinks + recent):
                raise ValueError(f"epure: sparse=(count, sinks, recent) with sinks + recent <= count (got {sparse})")
        self.sparse = sparse
        self._layers = [self.cache.layer(i) for i in range(decoder.layers)]
        # rows that the fused linears of a block take; larger batches go through linear_multi and separate glue
        rms, none = _native.PRO_RMSNORM, _native.PRO_NONE
        self._fused_rows = min(_native.decode_linear_max_rows(*call) for call in (
            (sh.hidden, rms, _native.EPI_STORE), (sh.hidden, rms, _native.EPI_SILU_MUL),
            (sh.heads * sh.head_dim, none, _native.EPI_RESIDUAL), (sh.intermediate, none, _native.EPI_RESIDUAL)
        )) if decoder._fusable else 0
        self._graphs = {}

    def _logits(self, h):
        """Float32 logits [rows, vocab] of the residual rows ``h``."""
        d = self.decoder
        y = _native.add_rmsnorm(h, eps=d.eps)
        if not d.fp32_logits:
            return F.linear(y, d.lm_head).float()
        if d.lm_head_f32 is None:
            d.lm_head_f32 = d.lm_head.float()
        return y.float() @ d.lm_head_f32.T

    def _write(self, pages, q, k, v, seq, pos):
        """q, k, v [rows, heads * head_dim] normed, rotated and written; q [rows, heads, head_dim]."""
        d, hd, rows = self.decoder, self.shapes.head_dim, q.shape[0]
        q = q.view(rows, -1, hd)
        return paged.write(pages, k.view(rows, -1, hd), v.view(rows, -1, hd), seq, pos, q=q, q_out=q, cos=d.cos,
                           sin=d.sin, qk_norm=d.qk_norm, eps=d.eps)

    def _attend(self, layer, pages, q, lengths, seq, first, scale, shared):
        """Attention of a step's rows q [rows, heads, head_dim]."""
        if shared is not None:
            return paged.attend_shared(pages, q, lengths, *shared, seq=seq, scale=scale)
        if self.sparse is None:
            return paged.attend(pages, q, lengths, seq=seq, scale=scale)
        count, sinks, recent = self.sparse
        bounds = self.cache.bounds[layer]
        paged.summarise(pages, bounds, lengths, seq=seq, first=first)
        chosen = paged.select(pages, bounds, q, lengths, count, seq=seq, sinks=sinks, recent=recent)
        return paged.attend(pages, q, lengths, seq=seq, scale=scale, blocks=chosen)

    # -- one token a row -----------------------------------------------------------------------------------------
    def step(self, tokens, seq, pos, shared=None):
        """Logits [batch, vocab] after feeding token ``tokens[b]`` (int64) as token ``pos[b]`` (int64) of sequence
        ``seq[b]`` (int32), all on the device.  A negative position is an idle row.  The pages must be reserved
        (``cache.reserve``).  Static shapes: capturable.

        Several rows may be tokens of one sequence (drafts): each attends over its own position and those before it.
        ``shared``: ``(starts, prefix)`` as ``paged.attend_shared`` takes them, for rows that have their first tokens in
        common; not with ``sparse``, where a call has one row a sequence."""
        if shared is not None and self.sparse is not None:
            raise ValueError("epure: a sparse step reads selected blocks, not a shared prefix")
        d, sh = self.decoder, self.shapes
        B, scale = tokens.shape[0], 1.0 / math.sqrt(sh.head_dim)
        lengths = (pos + 1).clamp_(min=0)                              # idle rows have no tokens
        first = pos.clamp(min=0) if self.sparse is not None else None
        h = d.embed[tokens]                                            # residual stream [B, hidden]
        fused = B <= self._fused_rows
        y = None if fused else _native.add_rmsnorm(h, eps=d.eps)
        for layer, (pages, b) in enumerate(zip(self._layers, d.stack.blocks)):
            qkv = [b["q_proj"], b["k_proj"], b["v_proj"]]
            if fused:
                q, k, v = _native.decode_linear(h, qkv, prologue=_native.PRO_RMSNORM, eps=d.eps)
            else:
                q, k, v = _native.linear_multi(y, qkv)
            q = self._write(pages, q, k, v, seq, pos)
            att = self._attend(layer, pages, q, lengths, seq, first, scale, shared).view(B, -1)
            if fused:
                _native.decode_linear(att, [b["o_proj"]], epilogue=_native.EPI_RESIDUAL, outs=[h])
                (a,) = _native.decode_linear(h, [b["gate_proj"], b["up_proj"]], prologue=_native.PRO_RMSNORM,
                                             epilogue=_native.EPI_SILU_MUL, eps=d.eps)
                _native.decode_linear(a, [b["down_proj"]], epilogue=_native.EPI_RESIDUAL, outs=[h])
            else:
                (o,) = _native.linear_multi(att, [b["o_proj"]])
                y = _native.add_rmsnorm(h, add=o, h_out=h, eps=d.eps)
                g, u = _native.linear_multi(y, [b["gate_proj"], b["up_proj"]])
                (o,) = _native.linear_multi(_native.silu_mul(g, u), [b["down_proj"]])
                y = _native.add_rmsnorm(h, add=o, h_out=h, eps=d.eps)  # the next layer's input norm
        return self._logits(h)

    # -- prompts -------------------------------------------------------------------------------------------------
    def prefill(self, seq, prompt, past=0):
        """Writes ``prompt`` (long [T]) as tokens past .. past + T - 1 of sequence ``seq`` and returns the logits
        [vocab] after its last token.  ``past`` > 0 continues a sequence (a prompt in chunks)."""
        d, sh, dev = self.decoder, self.shapes, self.device
        T, hd = prompt.shape[0], sh.head_dim
        if T < 1:
            raise ValueError("epure: an empty prompt")
        self.cache.reserve(seq, past + T)
        if self.sparse is not None:                                    # the bounds of the pages that the prompt fills
            row, till = torch.tensor([seq], dtype=torch.int32, device=dev), torch.tensor([past + T], device=dev)
            since = torch.tensor([past], device=dev)
        pos = torch.arange(past, past + T, device=dev)
        every = torch.arange(past + T, device=dev)
        ids = torch.full((past + T,), seq, dtype=torch.int32, device=dev)
        seen = None if past == 0 else every[None, :] <= pos[:, None]
        h = d.embed[prompt.to(dev)]
        for layer, (pages, b) in enumerate(zip(self._layers, d.stack.blocks)):
            q, k, v = _native.linear_multi(d._rms(h), [b["q_proj"], b["k_proj"], b["v_proj"]])
            q = self._write(pages, q, k, v, ids[past:], pos)
            if self.sparse is not None:
                paged.summarise(pages, self.cache.bounds[layer], till, seq=row, first=since)
            k, v = paged.read(pages, ids, every, dtype=d.dtype)
            att = F.scaled_dot_product_attention(q.transpose(0, 1)[None], k.transpose(0, 1)[None],
                                                 v.transpose(0, 1)[None], attn_mask=seen, is_causal=seen is None,
                                                 scale=1.0 / math.sqrt(hd), enable_gqa=True)
            att = att[0].transpose(0, 1).reshape(T, sh.heads * hd)
            h = h + _native.linear_multi(att, [b["o_proj"]])[0]
            g, u = _native.linear_multi(d._rms(h), [b["gate_proj"], b["up_proj"]])
            h = h + _native.linear_multi((F.silu(g.float()) * u.float()).to(d.dtype), [b["down_proj"]])[0]
        return self._logits(h[-1:].contiguous())[0]

    # -- greedy decoding -----------------------------------------------------------------------------------------
    def _captured(self, batch, behind=False):
        """(graph, tok, seq, pos, starts, prefix): one greedy step of ``batch`` rows, all of them behind one prefix where
        ``behind``; writes the argmax into tok, advances pos."""
        if (batch, behind) not in self._graphs:
            dev = self.device
            tok = torch.zeros(batch, dtype=torch.long, device=dev)
            seq = torch.arange(batch, dtype=torch.int32, device=dev)
            pos = torch.full((batch,), -1, dtype=torch.long, device=dev)     # idle rows: no cache is touched
            starts = torch.tensor([0, batch], dtype=torch.int32, device=dev)
            prefix = torch.zeros(1, dtype=torch.long, device=dev)
            shared = (starts, prefix) if behind else None

            def body():
                tok.copy_(torch.argmax(self.step(tok, seq, pos, shared), dim=-1))
                pos.add_(1)

            side = torch.cuda.Stream(device=dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                body()
            torch.cuda.current_stream(dev).wait_stream(side)
            pos.fill_(-1)
            torch.cuda.synchronize(dev)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                body()
            self._graphs[batch, behind] = (graph, tok, seq, pos, starts, prefix)
        return self._graphs[batch, behind]

    def _check(self, prompts):
        if not 1 <= len(prompts) <= self.cache.seqs:
            raise ValueError(f"epure: {len(prompts)} prompts for a cache of {self.cache.seqs} sequences")

    def _begin(self, prompts, n_new, prefix):
        """Reserves and fills the sequences of ``prompts`` (behind the common tokens ``prefix``, if any) with room for
        ``n_new`` more tokens: (logits behind each, lengths, tokens in common), the first a list of tensors."""
        n = 0 if prefix is None else prefix.shape[0]
        whole = 0
        logits, lengths = [], []
        for i, p in enumerate(prompts):
            if i == 0:
                self.cache.reserve(0, n + p.shape[0] + n_new)
                if n:
                    self.prefill(0, prefix)
                    whole = n // self.cache.page_size * self.cache.page_size
            elif n:                                        # the prefix's whole pages are shared, its rest is written again
                self.cache.share(i, 0, whole)
            self.cache.reserve(i, n + p.shape[0] + n_new)
            if n and i and whole < n:
                self.prefill(i, prefix[whole:], past=whole)
            logits.append(self.prefill(i, p, past=n))
            lengths.append(n + p.shape[0])
        return logits, lengths, n

    def generate(self, prompts, n_new, graph=True, prefix=None):
        """``n_new`` greedy tokens after each of the ``prompts`` (long tensors), a long tensor [len(prompts), n_new].
        ``prefix`` (a long tensor) comes before every prompt: it is computed and kept once, and each step's attention
        reads it once for all rows.  The sequences 0 .. len(prompts) - 1 are used and released."""
        self._check(prompts)
        B, dev = len(prompts), self.device
        out = torch.empty(B, n_new, dtype=torch.long, device=dev)
        try:
            logits, lengths, n = self._begin(prompts, n_new, prefix)
            tok, pos = torch.stack([torch.argmax(x) for x in logits]), torch.tensor(lengths, device=dev)
            seq = torch.arange(B, dtype=torch.int32, device=dev)
            behind = n > 0 and self.sparse is None
            if graph:
                g, gtok, gseq, gpos, _, gprefix = self._captured(B, behind)
                gtok.copy_(tok)
                gseq.copy_(seq)
                gpos.copy_(pos)
                gprefix.fill_(n)
                for t in range(n_new):
                    out[:, t] = gtok
                    if t + 1 < n_new:
                        g.replay()
            else:
                shared = (torch.tensor([0, B], dtype=torch.int32, device=dev), torch.tensor([n], device=dev)) if behind else None
                for t in range(n_new):
                    out[:, t] = tok
                    if t + 1 < n_new:
                        tok = torch.argmax(self.step(tok, seq, pos + t, shared), dim=-1)
        finally:
            for i in range(B):
                self.cache.release(i)
        return out

    # -- drafted tokens ------------------------------------------------------------------------------------------
    def judge(self, tokens, drafts, seq, pos, uniforms, temperature=1.0, draft_probs=None):
        """One pass over drafted tokens: ``tokens`` [batch] (the last known token of each sequence, at ``pos``) and
        ``drafts`` [batch, n] behind it (a row's end at its first one outside the vocabulary) are fed together, n + 1 rows
        a sequence that share what the sequence holds already, and judged by ``sampling.verify`` with the numbers ``uniforms``
        [batch, n + 1].  ``temperature`` 0 takes the most likely token.  Returns verify's ``(tokens [batch, n + 1],
        accepted [batch])``: a row's first ``accepted + 1`` tokens are its next ones.  The cache then holds ``pos +
        accepted + 1`` of its tokens; the last one returned is the next call's.  The pages must be reserved up to ``pos +
        n + 1`` tokens.  A negative position is an idle row.  Not with ``sparse``.  Capturable."""
        if self.sparse is not None:
            raise ValueError("epure: drafted tokens are judged over the whole cache (sparse=None)")
        B, n = drafts.shape
        dev = self.device
        drafts = drafts.masked_fill(drafts >= self.decoder.embed.shape[0], -1)
        rows = torch.cat((tokens[:, None], drafts), 1)
        there = (rows >= 0).to(torch.long).cumprod(1) * (pos >= 0)[:, None]
        step = torch.arange(n + 1, device=dev)
        at = torch.where(there > 0, pos[:, None] + step, -1)
        starts = torch.arange(0, B * (n + 1) + 1, n + 1, dtype=torch.int32, device=dev)
        logits = self.step(rows.clamp(min=0).reshape(-1), seq.repeat_interleave(n + 1), at.reshape(-1),
                           (starts, (pos + 1).clamp(min=0)))
        return sampling.verify(_probabilities(logits.view(B, n + 1, -1), temperature), draft_probs, drafts, uniforms)

    def speculate(self, prompts, n_new, drafts=4, temperature=0.0, prefix=None, generator=None):
        """``n_new`` tokens after each of the ``prompts``, drafted ``drafts`` at a time by looking the last two tokens up
        in what a sequence holds so far (the tokens behind their last occurrence), and the number of passes it took.
        ``temperature`` 0 gives ``generate``'s tokens but for near ties; ``generator`` (of the decoder's device) draws
        the random numbers otherwise.  A sequence needs room for ``drafts + 1`` tokens more."""
        self._check(prompts)
        B, dev = len(prompts), self.device
        if drafts < 0 or self.sparse is not None:
            raise ValueError(f"epure: drafts={drafts} (at least 0, and judged over the whole cache: sparse=None)")
        room = n_new + drafts + 1
        passes = 0
        try:
            logits, _, n = self._begin(prompts, room, prefix)
            u = torch.rand(B, 1, device=dev, generator=generator)
            none = torch.empty(B, 0, dtype=torch.long, device=dev)
            first, _ = sampling.verify(_probabilities(torch.stack(logits)[:, None], temperature), None, none, u)
            before = [] if prefix is None else prefix.tolist()
            text = [before + p.tolist() + [t] for p, t in zip(prompts, first[:, 0].tolist())]
            done = [n + p.shape[0] + n_new for p in prompts]
            seq = torch.arange(B, dtype=torch.int32, device=dev)
            while any(len(x) < d for x, d in zip(text, done)):
                guess = [_look_up(x, drafts) for x in text]
                pos = [len(x) - 1 if len(x) < d else -1 for x, d in zip(text, done)]
                u = torch.rand(B, drafts + 1, device=dev, generator=generator)
                got, kept = self.judge(torch.tensor([x[-1] for x in text], device=dev),
                                       torch.tensor(guess, dtype=torch.long, device=dev).view(B, drafts), seq,
                                       torch.tensor(pos, device=dev), u, temperature)
                passes += 1
                for x, p, tokens, k in zip(text, pos, got.tolist(), kept.tolist()):
                    if p >= 0:
                        x += tokens[:k + 1]
        finally:
            for i in range(B):
                self.cache.release(i)
        out = torch.tensor([x[d - n_new:d] for x, d in zip(text, done)], dtype=torch.long, device=dev).view(B, n_new)
        return out, passes


def _probabilities(logits, temperature):
    """What tokens are drawn with; a temperature of 0 takes the most likely one."""
    if temperature > 0:
        return torch.softmax(logits / temperature, -1)
    return torch.zeros_like(logits).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)


def _look_up(text, count):
    """Up to ``count`` tokens behind the last earlier occurrence of the text's last two, padded with -1."""
    last = text[-2:]
    for i in range(len(text) - 3, -1, -1):
        if text[i:i + 2] == last:
            got = text[i + 2:i + 2 + count]
            return got + [-1] * (count - len(got))
    return [-1] * count
