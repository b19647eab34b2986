"""Text generation on B200: prompt prefill + KV-cache decode steps.

Mirrors the reference's ``generate(params, prompt_ids, n_tokens, key,
temperature)`` (nlearn/model.py:449-465): same prompt trimming (keep the last
``max_seq - n_tokens`` prompt tokens), same output (prompt followed by the new
tokens), sampling from softmax(logits / temperature) (temperature 0 = greedy).
The reference re-runs the whole model over the full token buffer for every
new token (model.py:417-447); here the prompt is run once through the
training kernels (flash forward, fused-epilogue GEMMs), every layer's q|k|v
rows are kept as the KV cache, and each further token is one decode step:

    embed(tok, pos) -> per layer: LN + qkv GEMM (M = batch), decode attention
    (appends k|v at pos), proj GEMM + residual, LN + FFN up + bias + GELU,
    FFN down + bias + residual -> final LN + LM-head GEMM (f32 logits)
    -> sampler -> pos += 1

(each "LN + GEMM" is one kernel at batch <= 8: the small-M GEMM applies the
LayerNorm while staging its A operand).

The position lives in device memory, so one decode step is captured into a
CUDA graph once and replayed per token.  ``Decoder`` does this for a batch of
prompts of one length; ``PagedDecoder`` for rows that come and go with prompts
of any lengths, over a paged cache (``nlearn_b200.paged``), with penalties,
biases and masks on the logits (``nlearn_b200.kernels.logits``).  The random stream (seed, position,
row; for ``PagedDecoder`` the request in place of the row) is this library's own counter-based one (the
reference's JAX PRNG key is replaced by an integer seed).
"""
from __future__ import annotations

import functools

import numpy as np
import torch

from . import _lib
from ._lib import check, lib, ptr, stream_handle
from .kernels.gemm import gemm_ex
from .kernels.logits import process_logits
from .model import FlatParams, GPTConfig
from .paged import paged_decode_attention, paged_kv_write, update_block_tables


def _check_ids(ids: np.ndarray, vocab: int) -> None:
    """Refuses token ids that no row of the embedding belongs to (the kernels would read past it)."""
    if ids.size and (ids.min() < 0 or ids.max() >= vocab):
        raise ValueError(f"prompt ids must lie in [0, {vocab}), got {ids.min()} to {ids.max()}")


class _DecodeStep:
    """Static buffers of one decode step of `batch` rows and its layers around the attention."""

    def __init__(self, params: FlatParams, cfg: GPTConfig, batch: int, max_len: int | None):
        self.P, self.cfg, self.B = params, cfg, batch
        self.S = max_len or cfg.max_seq
        if self.S > cfg.max_seq:
            raise ValueError(f"max_len {self.S} exceeds the positional table ({cfg.max_seq})")
        B, D, F, Vp = batch, cfg.d_model, cfg.d_ff, cfg.vocab_padded
        dev = params.device
        bf = dict(device=dev, dtype=torch.bfloat16)
        self.tok = torch.zeros(B, device=dev, dtype=torch.int32)
        self.out = torch.zeros(B, self.S + 1, device=dev, dtype=torch.int32)
        self.x, self.x2, self.x3, self.h, self.o = (torch.empty(B, D, **bf) for _ in range(5))
        self.qkv = torch.empty(B, 3 * D, **bf)
        self.a, self.u = torch.empty(B, F, **bf), torch.empty(B, F, **bf)
        self.mean = torch.empty(B, device=dev, dtype=torch.float32)
        self.rstd = torch.empty_like(self.mean)
        self.logits = torch.empty(B, Vp, device=dev, dtype=torch.float32)
        self._fuse_ln = True  # LayerNorm folded into the small-M GEMM (batch <= 8)

    def _layers(self, attention):
        """From the embedded rows in ``x`` to the logits; ``attention(layer)``
        turns ``qkv`` into ``o``."""
        cfg, P = self.cfg, self.P
        x = self.x
        for layer in range(cfg.n_layers):
            pre = f"blocks.{layer}."
            self._ln_linear(x, P.f(pre + "ln1.g"), P.f(pre + "ln1.b"), P.p(pre + "wqkv"), self.qkv)
            attention(layer)
            gemm_ex(self.o, P.p(pre + "wo"), out=self.x2, epilogue=_lib.EPI_RESID, resid=x)
            self._ln_linear(self.x2, P.f(pre + "ln2.g"), P.f(pre + "ln2.b"), P.p(pre + "w1"), self.u,
                            epilogue=_lib.EPI_BIAS_GELU, bias=P.f(pre + "b1"), aux=self.a)
            gemm_ex(self.u, P.p(pre + "w2"), out=self.x3, epilogue=_lib.EPI_RESID, bias=P.f(pre + "b2"),
                    resid=self.x2)
            x = self.x3
        V = cfg.vocab
        self._ln_linear(x, P.f("lnf.g"), P.f("lnf.b"), P.p("head.w")[:, :V], self.logits[:, :V])

    def _ln(self, x, y, g, b, M):
        check(lib.nl_layernorm_fwd(ptr(x), ptr(g), ptr(b), ptr(y), ptr(self.mean if M == self.B else
                                                                          torch.empty(M, device=x.device)),
                                   ptr(self.rstd if M == self.B else torch.empty(M, device=x.device)), M,
                                   self.cfg.d_model, self.cfg.ln_eps, stream_handle()), "nl_layernorm_fwd")

    def _ln_linear(self, x, g, b, W, out, epilogue=_lib.EPI_STORE, bias=None, aux=None):
        """out = LayerNorm(x) . W (+ epilogue): one fused small-M kernel when the
        shape allows (batch <= 8), else LayerNorm then the GEMM."""
        if self._fuse_ln:
            dt = _lib.F32 if out.dtype == torch.float32 else _lib.BF16
            st = lib.nl_linear_ln_small(ptr(x), x.stride(0), ptr(g), ptr(b), self.cfg.ln_eps, ptr(W), W.stride(0),
                                        ptr(out), out.stride(0), dt, out.shape[0], out.shape[1], W.shape[0],
                                        epilogue, ptr(bias), ptr(aux), None, stream_handle())
            if st == 0:
                return
            if st != -1:  # anything but NL_ERR_SHAPE ("not a shape the fused kernel takes") is an error
                check(st, "nl_linear_ln_small")
            self._fuse_ln = False
        self._ln(x, self.h, g, b, self.B)
        gemm_ex(self.h, W, out=out, epilogue=epilogue, bias=bias, aux=aux)


class Decoder(_DecodeStep):
    """KV caches and the captured decode step for one batch size, all rows at
    one position; ``generate`` may be called repeatedly."""

    def __init__(self, params: FlatParams, cfg: GPTConfig, batch: int = 1, max_len: int | None = None):
        super().__init__(params, cfg, batch, max_len)
        dev = params.device
        self.cache = [torch.zeros(batch, self.S, 3 * cfg.d_model, device=dev, dtype=torch.bfloat16)
                      for _ in range(cfg.n_layers)]
        self.pos = torch.zeros(1, device=dev, dtype=torch.int32)
        nbytes = lib.nl_decode_workspace_bytes(batch, cfg.n_heads, self.S)
        self.ws = torch.zeros(nbytes, device=dev, dtype=torch.uint8)
        self._graph = None
        self._graph_key = None

    # ------------------------------------------------------------------ pieces
    def _head_and_sample(self, hf_rows, seed: int, temperature: float):
        V = self.cfg.vocab
        gemm_ex(hf_rows, self.P.p("head.w")[:, :V], out=self.logits[:, :V])
        self._sample(seed, temperature)

    def _sample(self, seed: int, temperature: float):
        V = self.cfg.vocab
        check(lib.nl_sample_tokens(ptr(self.logits), self.logits.stride(0), V, float(temperature), int(seed),
                                   ptr(self.pos), ptr(self.tok), ptr(self.out), self.out.stride(0), self.B,
                                   stream_handle()), "nl_sample_tokens")
        check(lib.nl_decode_advance(ptr(self.pos), stream_handle()), "nl_decode_advance")

    def prefill(self, prompt: torch.Tensor, seed: int, temperature: float):
        """Run the [B, P] prompt, fill the caches for positions 0..P-1, sample
        the token for position P; afterwards pos = P."""
        cfg, P = self.cfg, self.P
        B, Pl = prompt.shape
        D, H, F = cfg.d_model, cfg.n_heads, cfg.d_ff
        M = B * Pl
        dev = prompt.device
        tok = prompt.to(torch.int32).contiguous()
        self.out[:, :Pl] = tok
        x = torch.empty(M, D, device=dev, dtype=torch.bfloat16)
        check(lib.nl_embed_fwd(ptr(tok), ptr(P.p("wte")), ptr(P.p("wpe")), ptr(x), M, Pl, D, stream_handle()),
              "nl_embed_fwd")
        h = torch.empty_like(x)
        o = torch.empty_like(x)
        L = torch.empty(B * H, Pl, device=dev, dtype=torch.float32)
        qs = (3 * D, 64, Pl * 3 * D)
        os_ = (D, 64, Pl * D)
        for layer in range(cfg.n_layers):
            pre = f"blocks.{layer}."
            self._ln(x, h, P.f(pre + "ln1.g"), P.f(pre + "ln1.b"), M)
            qkv = gemm_ex(h, P.p(pre + "wqkv"), out_dtype=torch.bfloat16)
            self.cache[layer][:, :Pl].copy_(qkv.view(B, Pl, 3 * D))
            check(lib.nl_flash_attention_fwd_strided(ptr(qkv), ptr(qkv[:, D:]), ptr(qkv[:, 2 * D:]), *qs, ptr(o),
                                                     *os_, ptr(L), B, H, Pl, 64, stream_handle()), "attn fwd")
            x2 = gemm_ex(o, P.p(pre + "wo"), out_dtype=torch.bfloat16, epilogue=_lib.EPI_RESID, resid=x)
            self._ln(x2, h, P.f(pre + "ln2.g"), P.f(pre + "ln2.b"), M)
            a = torch.empty(M, F, device=dev, dtype=torch.bfloat16)
            u = gemm_ex(h, P.p(pre + "w1"), out_dtype=torch.bfloat16, epilogue=_lib.EPI_BIAS_GELU,
                        bias=P.f(pre + "b1"), aux=a)
            x = gemm_ex(u, P.p(pre + "w2"), out_dtype=torch.bfloat16, epilogue=_lib.EPI_RESID,
                        bias=P.f(pre + "b2"), resid=x2)
        self._ln(x, h, P.f("lnf.g"), P.f("lnf.b"), M)
        self.pos.fill_(Pl - 1)
        self._head_and_sample(h.view(B, Pl, D)[:, -1], seed, temperature)

    def _attention(self, layer: int):
        check(lib.nl_decode_attention(ptr(self.qkv), ptr(self.cache[layer]), ptr(self.o), ptr(self.pos), ptr(self.ws),
                                      self.ws.numel(), self.B, self.cfg.n_heads, self.S, 64, stream_handle()),
              "nl_decode_attention")

    def step(self, seed: int, temperature: float):
        """One decode step: the token in ``tok`` at position ``pos``."""
        P = self.P
        check(lib.nl_decode_embed(ptr(self.tok), ptr(self.pos), ptr(P.p("wte")), ptr(P.p("wpe")), ptr(self.x),
                                  self.B, self.cfg.d_model, stream_handle()), "nl_decode_embed")
        self._layers(self._attention)
        self._sample(seed, temperature)

    def capture(self, seed: int, temperature: float):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self.step(seed, temperature)
        self._graph, self._graph_key = g, (int(seed), float(temperature))

    # ------------------------------------------------------------------ API
    def generate(self, prompt_ids, n_tokens: int, seed: int = 0, temperature: float = 1.0,
                 use_graph: bool = True) -> np.ndarray:
        """[P] or [B, P] prompt ids -> [B, P' + n_tokens] (P' after trimming)."""
        p = np.asarray(prompt_ids)
        if n_tokens > 0:
            _check_ids(p, self.cfg.vocab)
        p = p.astype(np.int32)
        if p.ndim == 1:
            p = p[None]
        if p.shape[0] != self.B:
            raise ValueError(f"decoder built for batch {self.B}, prompt batch {p.shape[0]}")
        if n_tokens <= 0:
            return p
        if n_tokens >= self.S:
            raise ValueError(f"n_tokens {n_tokens} must be below max_len {self.S}")
        if p.shape[1] + n_tokens > self.S:  # keep the most recent prompt tokens (model.py:462-463)
            p = p[:, -(self.S - n_tokens):]
        Pl = p.shape[1]
        self.prefill(torch.from_numpy(p).to(self.P.device), seed, temperature)
        for i in range(1, n_tokens):
            if use_graph and i >= 2:
                if self._graph is None or self._graph_key != (int(seed), float(temperature)):
                    self.capture(seed, temperature)
                self._graph.replay()
            else:
                self.step(seed, temperature)
        return self.out[:, :Pl + n_tokens].cpu().numpy()


def _on_device(method):
    """Run a method with the decoder's device current."""
    @functools.wraps(method)
    def run(self, *args, **kw):
        with torch.cuda.device(self.P.device):
            return method(self, *args, **kw)
    return run


class PagedDecoder(_DecodeStep):
    """Generation for rows that come and go, each with a prompt, a length and
    rules of its own, over a paged KV cache.

    ``add`` admits a prompt to a free row, ``step`` draws a token for every row
    in use (one captured CUDA graph), ``tokens`` reads a row, ``release`` gives its
    pages back; ``generate`` runs any number of prompts through the rows.  A
    step whose rows all fit is never refused: the host keeps count of the pages.

    Prompts are numbered in the order of their admission (``next_request`` is the
    next one's number), and a token's random bits depend on (seed, position,
    number): prompts that use a row one after the other draw independently,
    whichever rows they get, and a new decoder given the same prompts repeats the draws.

    cache_dtype bfloat16, or float8_e4m3fn (half the bytes; keys and values
    are stored as they are, scale 1).
    """

    MAX_GRAPHS = 32

    def __init__(self, params: FlatParams, cfg: GPTConfig, max_batch: int = 8, n_pages: int | None = None,
                 page_size: int = 16, max_len: int | None = None, max_bias: int = 32, seed: int = 0,
                 temperature: float = 1.0, cache_dtype=torch.bfloat16):
        super().__init__(params, cfg, max_batch, max_len)
        R, H, dev = max_batch, cfg.n_heads, params.device
        if page_size < 1 or max_bias < 0 or max_batch < 1 or (n_pages is not None and n_pages < 1):
            raise ValueError(f"page_size {page_size}, max_bias {max_bias}, max_batch {max_batch}, n_pages {n_pages}: "
                             "out of range")
        self.page_size, self.seed, self.temperature = page_size, int(seed), float(temperature)
        self.blocks = -(-self.S // page_size)
        self.n_pages = R * self.blocks if n_pages is None else n_pages
        i32, f32 = dict(device=dev, dtype=torch.int32), dict(device=dev, dtype=torch.float32)
        shape = (self.n_pages, H, page_size, 64)
        self.k_cache, self.v_cache = ([torch.zeros(shape, device=dev, dtype=torch.bfloat16).to(cache_dtype)
                                       for _ in range(cfg.n_layers)] for _ in range(2))
        self.block_table = torch.full((R, self.blocks), -1, **i32)
        self.lens = torch.zeros(R, **i32)          # tokens of a row; its cache holds their keys after a step
        self.free_pages = torch.arange(self.n_pages, **i32)
        self.n_free = torch.full((1,), self.n_pages, **i32)
        self.new = torch.zeros(R, **i32)           # 1: the row is in use
        self.now = torch.zeros(R, **i32)           # lengths of the rows that draw a token
        self.prompt_lens = torch.zeros(R, **i32)
        self.requests = torch.zeros(R, **i32)      # 32 bits of the number of the prompt a row was admitted with
        self.next_request = 0
        self.repetition, self.frequency, self.presence = torch.ones(R, **f32), torch.zeros(R, **f32), torch.zeros(R,
                                                                                                                 **f32)
        self.bias_ids, self.bias = torch.full((R, max_bias), -1, **i32), torch.zeros(R, max_bias, **f32)
        self.mask = torch.zeros(R, (cfg.vocab + 31) // 32, **i32)
        self.mask_rows = torch.full((R,), -1, **i32)
        self._len = [0] * R                        # host's copy of the lengths
        self._rules = [frozenset()] * R
        self._graphs = {}

    # ------------------------------------------------------------------ pieces
    def _pages(self, n: int) -> int:
        return -(-n // self.page_size)

    def free_rows(self) -> list[int]:
        return [r for r in range(self.B) if self._len[r] == 0]

    def free_page_count(self) -> int:
        # (a row's last token has no key in the cache until the next step)
        return self.n_pages - sum(self._pages(n - 1) for n in self._len if n)

    def _attention(self, layer: int):
        D, H = self.cfg.d_model, self.cfg.n_heads
        q, k, v = (self.qkv[:, i * D:(i + 1) * D].view(self.B, H, 64) for i in range(3))
        paged_decode_attention(q, self.k_cache[layer], self.v_cache[layer], self.block_table, self.lens, k, v,
                               out=self.o.view(self.B, H, 64))

    def _draw(self, lens, rules):
        """Rules, then a token for every row with lens > 0 (its tokens so far)."""
        V = self.cfg.vocab
        kw = {}
        if "penalties" in rules:
            kw.update(tokens=self.out, lens=lens, prompt_lens=self.prompt_lens, repetition=self.repetition,
                      frequency=self.frequency, presence=self.presence)
        if "bias" in rules:
            kw.update(bias_ids=self.bias_ids, bias=self.bias)
        if "mask" in rules:
            kw.update(mask=self.mask, mask_rows=self.mask_rows)
        if kw:
            process_logits(self.logits[:, :V], out=self.logits[:, :V], **kw)
        check(lib.nl_sample_tokens_requests(ptr(self.logits), self.logits.stride(0), V, self.temperature, self.seed,
                                            ptr(lens), ptr(self.requests), ptr(self.tok), ptr(self.out),
                                            self.out.stride(0), self.B, stream_handle()),
              "nl_sample_tokens_requests")

    def _embed(self, tok, lens, x):
        P, cfg = self.P, self.cfg
        check(lib.nl_decode_embed_rows(ptr(tok), ptr(lens), ptr(P.p("wte")), ptr(P.p("wpe")), ptr(x), tok.numel(),
                                       cfg.d_model, self.S, cfg.vocab, stream_handle()), "nl_decode_embed_rows")

    def _step(self, rules):
        update_block_tables(self.block_table, self.lens, self.new, self.free_pages, self.n_free, self.page_size,
                            self.B, lens_out=self.lens, n_free_out=self.n_free)
        self._embed(self.tok, self.lens, self.x)
        self._layers(self._attention)
        self._draw(self.lens, rules)

    def _run_step(self, rules, use_graph):
        if not use_graph:
            return self._step(rules)
        key = (rules, self.seed, self.temperature)
        graph = self._graphs.pop(key, None)
        if graph is None:
            self._step(rules)  # (the first step of a kind runs eagerly: it sets the kernels up)
            self._keep_graph(key, False)
            return
        if graph is False:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self._step(rules)
        self._keep_graph(key, graph)  # (after the capture has succeeded)
        graph.replay()

    def _keep_graph(self, key, graph):
        """Keep the MAX_GRAPHS graphs used last (a seed and temperature have up to 8, one for each set of rules)."""
        self._graphs[key] = graph
        if len(self._graphs) > self.MAX_GRAPHS:
            torch.cuda.synchronize()  # (it may still run, on any stream)
            del self._graphs[next(iter(self._graphs))]

    def _set_rules(self, row, repetition, frequency, presence, bias, allowed):
        rules = set()
        if repetition != 1.0 or frequency != 0.0 or presence != 0.0:
            rules.add("penalties")
        self.repetition[row], self.frequency[row], self.presence[row] = repetition, frequency, presence
        self.bias_ids[row] = -1
        if bias:
            ids = list(bias)
            if len(ids) > self.bias_ids.shape[1]:
                raise ValueError(f"{len(ids)} biases, over max_bias {self.bias_ids.shape[1]}")
            self.bias_ids[row, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
            self.bias[row, :len(ids)] = torch.tensor([float(bias[i]) for i in ids])
            rules.add("bias")
        self._set_allowed(row, allowed)
        if allowed is not None:
            rules.add("mask")
        self._rules[row] = frozenset(rules)

    def _run_prompts(self, rows, sizes, flat, plan):
        """The prompts through the layers into their slots, and the first token of each."""
        cfg, P, D, H, F = self.cfg, self.P, self.cfg.d_model, self.cfg.n_heads, self.cfg.d_ff
        dev, T = self.P.device, sum(sizes)
        at = [sum(sizes[:i]) for i in range(len(sizes))]
        for row, a, n in zip(rows, at, sizes):
            self.out[row, :n] = flat[a:a + n]
            self.prompt_lens[row] = n
        x = torch.empty(T, D, device=dev, dtype=torch.bfloat16)
        self._embed(flat, plan.positions + 1, x)
        h, o = torch.empty_like(x), torch.empty_like(x)
        L = torch.empty(H, max(sizes), device=dev, dtype=torch.float32)
        for layer in range(cfg.n_layers):
            pre = f"blocks.{layer}."
            self._ln(x, h, P.f(pre + "ln1.g"), P.f(pre + "ln1.b"), T)
            qkv = gemm_ex(h, P.p(pre + "wqkv"), out_dtype=torch.bfloat16)
            q, k, v = (qkv[:, i * D:(i + 1) * D] for i in range(3))
            paged_kv_write(k.view(T, H, 64), v.view(T, H, 64), self.k_cache[layer], self.v_cache[layer], plan.slots)
            for a, n in zip(at, sizes):  # (kernels on one stream: L may serve all)
                check(lib.nl_flash_attention_fwd_strided(ptr(q[a:]), ptr(k[a:]), ptr(v[a:]), 3 * D, 64, n * 3 * D,
                                                         ptr(o[a:]), D, 64, n * D, ptr(L), 1, H, n, 64,
                                                         stream_handle()), "attn fwd")
            x2 = gemm_ex(o, P.p(pre + "wo"), out_dtype=torch.bfloat16, epilogue=_lib.EPI_RESID, resid=x)
            self._ln(x2, h, P.f(pre + "ln2.g"), P.f(pre + "ln2.b"), T)
            a_ = torch.empty(T, F, device=dev, dtype=torch.bfloat16)
            u = gemm_ex(h, P.p(pre + "w1"), out_dtype=torch.bfloat16, epilogue=_lib.EPI_BIAS_GELU,
                        bias=P.f(pre + "b1"), aux=a_)
            x = gemm_ex(u, P.p(pre + "w2"), out_dtype=torch.bfloat16, epilogue=_lib.EPI_RESID,
                        bias=P.f(pre + "b2"), resid=x2)
        last = torch.tensor([a + n - 1 for a, n in zip(at, sizes)], device=dev)
        where = torch.tensor(rows, device=dev)
        self.x3.zero_()
        self.x3[where] = x[last]
        V = cfg.vocab
        self._ln_linear(self.x3, P.f("lnf.g"), P.f("lnf.b"), P.p("head.w")[:, :V], self.logits[:, :V])
        self.now.zero_()
        self.now[where] = self.lens[where]
        numbers = (self.next_request + np.arange(len(rows))) & 0xFFFFFFFF
        self.requests[where] = torch.from_numpy(numbers.astype(np.uint32).view(np.int32)).to(dev)
        self._draw(self.now, frozenset().union(*(self._rules[r] for r in rows)))
        self.new[where] = 1
        self.next_request += len(rows)

    # ------------------------------------------------------------------ API
    def set_allowed(self, row: int, allowed) -> None:
        """Token ids that a row in use may draw from now on (None: all; a grammar calls this between steps)."""
        if not 0 <= row < self.B or not self._len[row]:
            raise ValueError(f"row {row} is not in use")
        self._set_allowed(row, allowed)

    def _set_allowed(self, row, allowed):
        if allowed is None:
            self.mask_rows[row] = -1
            self._rules[row] = self._rules[row] - {"mask"}
            return
        ids = np.asarray(list(allowed), np.int64)
        if not ids.size or ids.min() < 0 or ids.max() >= self.cfg.vocab:
            raise ValueError("allowed must name at least one token, all inside the vocabulary")
        words = np.zeros(self.mask.shape[1], np.uint32)
        np.bitwise_or.at(words, ids // 32, np.uint32(1) << (ids % 32).astype(np.uint32))
        self.mask[row] = torch.from_numpy(words.view(np.int32)).to(self.mask.device)
        self.mask_rows[row] = row
        self._rules[row] = self._rules[row] | {"mask"}

    @_on_device
    def add(self, prompts, *, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0,
            bias: dict | None = None, allowed=None) -> list[int]:
        """Admit prompts (a list of 1-D id arrays) to free rows, run them and
        draw the first token of each; -> the rows.  The rules (see
        ``process_logits``) hold for all of them; ``allowed`` is a set of token ids."""
        prompts = [np.asarray(p).reshape(-1) for p in prompts]
        for p in prompts:
            _check_ids(p, self.cfg.vocab)
        allowed = None if allowed is None else list(allowed)  # (read once for each row)
        rows = self.free_rows()[:len(prompts)]
        if len(rows) < len(prompts):
            raise RuntimeError(f"{len(prompts)} prompts, {len(rows)} free rows")
        sizes = [p.size for p in prompts]
        if any(n < 1 or n >= self.S for n in sizes):
            raise ValueError(f"prompt lengths {sizes}: must be 1 to {self.S - 1}")
        if sum(self._pages(n) for n in sizes) > self.free_page_count():
            raise RuntimeError(f"prompts need {sum(self._pages(n) for n in sizes)} pages, {self.free_page_count()} free")
        if not rows:
            return rows
        dev, T = self.P.device, sum(sizes)
        # the flat list holds the prompts in the order of their rows, which is ascending
        flat = torch.from_numpy(np.concatenate(prompts).astype(np.int32)).to(dev)
        for row in rows:
            self._set_rules(row, repetition, frequency, presence, bias, allowed)
        grow = torch.zeros(self.B, dtype=torch.int32)
        grow[rows] = torch.tensor(sizes, dtype=torch.int32)
        grow = grow.to(dev)
        for row, n in zip(rows, sizes):
            self._len[row] = n
        try:
            plan = update_block_tables(self.block_table, self.lens, grow, self.free_pages, self.n_free, self.page_size,
                                       T, lens_out=self.lens, n_free_out=self.n_free)
            self._run_prompts(rows, sizes, flat, plan)
        except BaseException:
            self.release(rows)  # (whether or not the device has given them their pages)
            raise
        for row in rows:
            self._len[row] += 1
        return rows

    @_on_device
    def step(self, n: int = 1, use_graph: bool = True) -> None:
        """Draw n tokens for every row in use."""
        for _ in range(n):
            used = [r for r in range(self.B) if self._len[r]]
            if not used:
                return
            if any(self._len[r] > self.S for r in used):
                raise RuntimeError(f"a row is at its full length of {self.S} tokens: release it")
            grow = sum(self._pages(self._len[r]) - self._pages(self._len[r] - 1) for r in used)
            if grow > self.free_page_count():
                raise RuntimeError(f"the step needs {grow} pages, {self.free_page_count()} free: release a row")
            rules = frozenset().union(*(self._rules[r] for r in used))
            try:
                self._run_step(rules, use_graph)
            except BaseException:
                # back to before the step: the pages it took are still on the stack, above its size
                last = torch.tensor([max(0, n - 1) for n in self._len], device=self.P.device)
                self.lens.copy_(last)
                self.n_free.fill_(self.free_page_count())
                self.tok.copy_(self.out.gather(1, last[:, None])[:, 0])
                raise
            for r in used:
                self._len[r] += 1

    def tokens(self, row: int) -> np.ndarray:
        """The row's prompt and the tokens drawn so far."""
        return self.out[row, :self._len[row]].cpu().numpy()

    @_on_device
    def release(self, rows) -> None:
        """End rows: their pages are free, the rows may be admitted anew."""
        rows = list(rows)  # (walked twice)
        done = torch.zeros(self.B, dtype=torch.int32)
        for r in rows:
            if not self._len[r]:
                raise ValueError(f"row {r} is not in use")
            done[r] = 1
        done = done.to(self.P.device)
        update_block_tables(self.block_table, self.lens, torch.zeros_like(self.new), self.free_pages, self.n_free,
                            self.page_size, 0, done=done, lens_out=self.lens, n_free_out=self.n_free)
        for r in rows:
            self._len[r] = 0
            self._rules[r] = frozenset()
            self.new[r] = 0
            self.mask_rows[r] = -1
            self.bias_ids[r] = -1
            self.repetition[r], self.frequency[r], self.presence[r] = 1.0, 0.0, 0.0

    def generate(self, prompts, n_tokens, use_graph: bool = True, **rules) -> list[np.ndarray]:
        """Prompts of any lengths and number, n_tokens (one number, or one per prompt)
        drawn for each: as rows and pages come free the next prompts are admitted.
        Long prompts keep their last ids, as in ``Decoder``."""
        if any(self._len):
            raise RuntimeError("generate needs all rows free")
        if rules.get("allowed") is not None:
            rules["allowed"] = list(rules["allowed"])  # (read by every admission)
        prompts = [np.asarray(p).reshape(-1) for p in prompts]
        counts = [int(n) for n in np.broadcast_to(n_tokens, (len(prompts),))]
        for p, n in zip(prompts, counts):
            if n > 0:
                _check_ids(p, self.cfg.vocab)
        prompts = [p.astype(np.int32) for p in prompts]
        if any(n >= self.S for n in counts):
            raise ValueError(f"n_tokens {max(counts)} must be below max_len {self.S}")
        if any(p.size < 1 for p, n in zip(prompts, counts) if n > 0):
            raise ValueError("an empty prompt")
        prompts = [p[-(self.S - n):] if n > 0 else p for p, n in zip(prompts, counts)]
        done: list = [p.copy() if n <= 0 else None for p, n in zip(prompts, counts)]
        queue = [i for i in range(len(prompts)) if done[i] is None]
        running: dict[int, int] = {}
        need = lambda i: self._pages(prompts[i].size + counts[i] - 1)  # noqa: E731  (the last token's key is never kept)
        for i in queue:
            if need(i) > self.n_pages:
                raise ValueError(f"prompt {i} needs {need(i)} pages, the cache has {self.n_pages}")
        try:
            while queue or running:
                take, held = [], sum(need(i) for i in running.values())
                for i in queue[:len(self.free_rows())]:
                    if held + need(i) > self.n_pages:
                        break
                    held += need(i)
                    take.append(i)
                if take:
                    del queue[:len(take)]
                    running.update(zip(self.add([prompts[i] for i in take], **rules), take))
                left = {r: prompts[i].size + counts[i] - self._len[r] for r, i in running.items()}
                if min(left.values()) > 0:
                    self.step(min(left.values()), use_graph)
                ended = [r for r, n in left.items() if n == min(left.values())]
                for r in ended:
                    done[running.pop(r)] = self.tokens(r)
                self.release(ended)
        except BaseException:
            self.release(r for r in range(self.B) if self._len[r])  # (all rows were free at the start)
            raise
        return done


def generate(trainer_or_params, prompt_ids, n_tokens, seed: int = 0, temperature: float = 1.0,
             cfg: GPTConfig | None = None, **rules):
    """Reference-shaped entry point: a Trainer (or FlatParams + cfg), a 1-D or
    [B, P] prompt -> tokens (1-D for a 1-D prompt).  A list of prompts of
    different lengths, an n_tokens per prompt, or any of the rules of
    ``PagedDecoder.add`` (repetition, frequency, presence, bias, allowed) run on the
    paged cache; a list of prompts, or an n_tokens for each, then gives a list of
    arrays, a [B, P] array with one n_tokens a [B, P + n_tokens] one."""
    P = getattr(trainer_or_params, "P", trainer_or_params)
    cfg = cfg or getattr(trainer_or_params, "cfg", None) or P.cfg
    several = isinstance(prompt_ids, (list, tuple)) and any(np.ndim(p) == 1 for p in prompt_ids)
    if rules or np.ndim(n_tokens) or (several and len({len(p) for p in prompt_ids}) > 1):
        prompts = prompt_ids if several or np.ndim(prompt_ids) == 2 else [prompt_ids]
        dec = PagedDecoder(P, cfg, max_batch=max(1, min(len(prompts), 32)), max_bias=len(rules.get("bias") or ()),
                           seed=seed, temperature=temperature)
        out = dec.generate(prompts, n_tokens, **rules)
        if several or np.ndim(prompt_ids) == 2:
            return out if several or np.ndim(n_tokens) or not out else np.stack(out)
        return out[0]
    p = np.asarray(prompt_ids)
    dec = Decoder(P, cfg, batch=1 if p.ndim == 1 else p.shape[0])
    out = dec.generate(p, n_tokens, seed, temperature)
    return out[0] if p.ndim == 1 else out
