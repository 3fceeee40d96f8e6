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
"""
import math

import torch
import torch.nn.functional as F

from . import _native, paged


class BatchDecoder:
    """``decoder``: a ``PackedDecoder`` in mode "ours" (its stores, embedding, lm_head and rotary tables are used, its
    own cache is not).  ``seqs`` sequences of up to the decoder's ``max_len`` tokens; ``pages`` defaults to room for
    all of them.  ``format``: "same", "int8" or "fp8"."""

    def __init__(self, decoder, seqs=16, format="same", page_size=64, pages=None):
        if decoder.mode != "ours" or decoder.dtype != torch.bfloat16:
            raise ValueError("epure: a BatchDecoder needs a PackedDecoder in linear_mode 'ours'")
        sh = decoder.shapes
        self.decoder, self.shapes, self.device = decoder, sh, decoder.device
        per_seq = -(-decoder.max_len // page_size)
        self.cache = paged.PagedKVCache(decoder.layers, pages or seqs * per_seq, page_size, sh.kv_heads, sh.head_dim,
                                        seqs, decoder.max_len, format, decoder.dtype, decoder.device)
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

    # -- one token a sequence ------------------------------------------------------------------------------------
    def step(self, tokens, seq, pos):
        """Logits [batch, vocab] after feeding token ``tokens[b]`` (int64) as token ``pos[b]`` (int64) of sequence
        ``seq[b]`` (int32), all on the device.  A negative position is an idle row.  The pages must be reserved
        (``cache.reserve``).  Static shapes: capturable."""
        d, sh = self.decoder, self.shapes
        B, scale = tokens.shape[0], 1.0 / math.sqrt(sh.head_dim)
        lengths = (pos + 1).clamp_(min=0)                              # idle rows have no tokens
        h = d.embed[tokens]                                            # residual stream [B, hidden]
        fused = B <= self._fused_rows
        y = None if fused else _native.add_rmsnorm(h, eps=d.eps)
        for pages, b in zip(self._layers, d.stack.blocks):
            qkv = [b["q_proj"], b["k_proj"], b["v_proj"]]
            if fused:
                q, k, v = _native.decode_linear(h, qkv, prologue=_native.PRO_RMSNORM, eps=d.eps)
            else:
                q, k, v = _native.linear_multi(y, qkv)
            q = self._write(pages, q, k, v, seq, pos)
            att = paged.attend(pages, q, lengths, seq=seq, scale=scale).view(B, -1)
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
        pos = torch.arange(past, past + T, device=dev)
        every = torch.arange(past + T, device=dev)
        ids = torch.full((past + T,), seq, dtype=torch.int32, device=dev)
        seen = None if past == 0 else every[None, :] <= pos[:, None]
        h = d.embed[prompt.to(dev)]
        for pages, b in zip(self._layers, d.stack.blocks):
            q, k, v = _native.linear_multi(d._rms(h), [b["q_proj"], b["k_proj"], b["v_proj"]])
            q = self._write(pages, q, k, v, ids[past:], pos)
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
    def _captured(self, batch):
        """(graph, tok, seq, pos): one greedy step of ``batch`` rows; writes the argmax into tok, advances pos."""
        if batch not in self._graphs:
            dev = self.device
            tok = torch.zeros(batch, dtype=torch.long, device=dev)
            seq = torch.arange(batch, dtype=torch.int32, device=dev)
            pos = torch.full((batch,), -1, dtype=torch.long, device=dev)     # idle rows: no cache is touched

            def body():
                tok.copy_(torch.argmax(self.step(tok, seq, pos), dim=-1))
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
            self._graphs[batch] = (graph, tok, seq, pos)
        return self._graphs[batch]

    def generate(self, prompts, n_new, graph=True):
        """``n_new`` greedy tokens after each of the ``prompts`` (long tensors), a long tensor [len(prompts), n_new].
        The sequences 0 .. len(prompts) - 1 are used and released."""
        B, dev = len(prompts), self.device
        if not 1 <= B <= self.cache.seqs:
            raise ValueError(f"epure: {B} prompts for a cache of {self.cache.seqs} sequences")
        out = torch.empty(B, n_new, dtype=torch.long, device=dev)
        try:
            first = []
            for i, p in enumerate(prompts):
                self.cache.reserve(i, p.shape[0] + n_new)
                first.append(torch.argmax(self.prefill(i, p)))
            tok, pos = torch.stack(first), torch.tensor([p.shape[0] for p in prompts], device=dev)
            seq = torch.arange(B, dtype=torch.int32, device=dev)
            if graph:
                g, gtok, gseq, gpos = self._captured(B)
                gtok.copy_(tok)
                gseq.copy_(seq)
                gpos.copy_(pos)
                for t in range(n_new):
                    out[:, t] = gtok
                    if t + 1 < n_new:
                        g.replay()
            else:
                for t in range(n_new):
                    out[:, t] = tok
                    if t + 1 < n_new:
                        tok = torch.argmax(self.step(tok, seq, pos + t), dim=-1)
        finally:
            for i in range(B):
                self.cache.release(i)
        return out
