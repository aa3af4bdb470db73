"""GPT-2 served from a paged key/value cache: requests of different lengths together,
greedy or by beam search, every Linear an int8 MatMulQ.

Where DeviceDecoder (gpt2.py) keeps a batch at one position over contiguous caches, as
the reference's KVDecoder does for one sequence (tools/run_gpt2.cpp:88-191), here the
prompts are packed one after another and every request has its own length. A pass over new
tokens -- a prompt, a chunk of one, or one token for every beam -- is the same sequence of
launches: LayerNorm, the fused QKV product, `serving.paged_attention` (which stores the new
keys and values in the pages and attends to all of the request's), the output product with
its residual, LayerNorm, and the two FFN products. `serving.beam_select` then chooses the
next tokens and `serving.beam_reorder` moves the cache along with the beams. One decoding
step is captured as a CUDA graph and replayed: lengths, page numbers, scores and tokens live
in device memory.

The cache holds f32 in mode "fp32" and bf16 in mode "bf16" (whose attention then returns
bf16 rows, the type that mode's products round their input to anyway).
"""
from __future__ import annotations

import itertools

import numpy as np
import torch

from . import serving
from ._lib import MAX_BATCH, MAX_BEAMS, check, lib
from .gpt2 import GPT2Weights
from .matmulq import PackedWeight, Workspace, matmul_q8


def assign_pages(prompt_lens, beams: int, max_new: int, page_size: int):
    """Which pages the beams read at first and which only they write: (table, owned, pages
    in all), both [requests * beams, columns]. A request's beams share its prompt's full
    pages (only the prompt's pass writes those); of the later columns each has its own, and
    reads its first beam's, where the prompt's last tokens are, until beams part."""
    width = max(-(-(p + max_new) // page_size) for p in prompt_lens)
    table, owned, count = [], [], 0
    for p in prompt_lens:
        shared = list(range(count, count + p // page_size))
        count += len(shared)
        first = None
        for _ in range(beams):
            mine = shared + list(range(count, count + width - len(shared)))
            count += width - len(shared)
            first = first or mine
            owned.append(mine)
            table.append(first)
    return np.array(table, np.int32), np.array(owned, np.int32), count


class PagedDecoder:
    """Serves GPT-2 weights (gpt2.GPT2Weights) on one GPU; see the module's docstring."""

    def __init__(self, w: GPT2Weights, mode: str = "fp32", page_size: int = 32, device="cuda"):
        cfg = w.cfg
        if page_size not in (16, 32, 64, 128):
            raise ValueError("page_size is 16, 32, 64 or 128")
        if mode not in ("fp32", "bf16"):
            raise ValueError("mode is 'fp32' or 'bf16'")
        self.cfg, self.mode, self.page_size = cfg, mode, page_size
        self.dev = torch.device(device)
        self.cache_dtype = torch.float32 if mode == "fp32" else torch.bfloat16
        f32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)
        pk = lambda qs: PackedWeight.from_int8(torch.from_numpy(qs[0]), torch.from_numpy(qs[1]), self.dev)
        self.wte, self.wpe = f32(w.wte), f32(w.wpe)
        self.layers = [{k: pk(v) if k in ("qkv", "o", "fc", "proj") else
                        tuple(f32(x) for x in v) if isinstance(v, tuple) else f32(v) for k, v in L.items()}
                       for L in w.layers]
        self.ln_f = tuple(f32(x) for x in w.ln_f)
        self.lm_head = pk(w.lm_head)
        self.ws, self.attn_ws = Workspace(self.dev), Workspace(self.dev)

    # -- pieces of a pass --------------------------------------------------------------
    def _layernorm(self, x, ln):
        y = torch.empty_like(x)
        check(lib().mtrtq_layernorm(x.data_ptr(), ln[0].data_ptr(), ln[1].data_ptr(), y.data_ptr(), x.shape[0],
                                    x.shape[1], self.cfg.eps, torch.cuda.current_stream(self.dev).cuda_stream),
              "mtrtq_layernorm")
        return y

    def _mm(self, x, w, bias=None, out=None, epilogue="none", residual=None):
        return matmul_q8(x, w, bias, out=out, mode=self.mode, workspace=self.ws, epilogue=epilogue, residual=residual)

    def _pass(self, tokens, positions, attend):
        """Hidden rows of `tokens` at `positions` (device, one entry per row) after every
        layer; attend(layer, q, k, v) gives a layer's attention rows."""
        cfg = self.cfg
        H, hd, D = cfg.n_head, cfg.head_dim, cfg.d_model
        x = self.wte[tokens] + self.wpe[positions]
        for i, ly in enumerate(self.layers):
            qkv = self._mm(self._layernorm(x, ly["ln1"]), ly["qkv"], ly["bqkv"])
            q, k, v = (t.view(-1, H, hd) for t in qkv.split(D, dim=1))
            a = attend(i, q, k, v).view(-1, D)
            self._mm(a, ly["o"], ly["bo"], out=x, epilogue="residual", residual=x)
            h = self._mm(self._layernorm(x, ly["ln2"]), ly["fc"], ly["bfc"], epilogue="gelu")
            self._mm(h, ly["proj"], ly["bproj"], out=x, epilogue="residual", residual=x)
        return x

    def _logits(self, x, out=None):
        return self._mm(self._layernorm(x, self.ln_f), self.lm_head, out=out)

    def _packed(self, prompts):
        lens = [len(p) for p in prompts]
        if not lens or min(lens) < 1 or max(lens) > self.cfg.n_pos:
            raise ValueError(f"every prompt has 1 to {self.cfg.n_pos} tokens")
        ids = np.concatenate([np.asarray(p, np.int64) for p in prompts])
        if ids.min() < 0 or ids.max() >= self.cfg.vocab:
            raise ValueError("a token id is outside the vocabulary")
        at = np.concatenate([np.arange(n) for n in lens])
        i32 = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32, device=self.dev)
        return lens, torch.from_numpy(ids).to(self.dev), torch.from_numpy(at).to(self.dev), \
            i32([0, *itertools.accumulate(lens)]), i32

    # -- public -----------------------------------------------------------------------
    def logits(self, prompts) -> list:
        """The next-token logits at every position of every prompt (for scoring: nothing is
        cached), in one packed pass: a float32 [len, vocab] tensor for each prompt."""
        lens, ids, at, cu, _ = self._packed(prompts)
        attend = lambda i, q, k, v: serving.prompt_attention(q, k, v, cu, out_dtype=self.cache_dtype,
                                                             workspace=self.attn_ws)
        return list(self._logits(self._pass(ids, at, attend)).split(lens))

    def generate(self, prompts, max_new: int, beams: int = 1, eos: int = -1, chunk: int | None = None,
                 use_graph: bool = True) -> dict:
        """Continues each prompt (a sequence of token ids, of any lengths) by max_new tokens:
        greedily, or by beam search with `beams` > 1; a beam that takes `eos` ends there (the
        rest of its row is eos). chunk: tokens of a prompt that one pass takes (all of
        them by default). Returns {"tokens": int32 [requests, beams, max_new], "scores":
        float32 [requests, beams] sums of log-probabilities}, best beam first."""
        lens, _, _, _, i32 = self._packed(prompts)
        if max_new < 1 or max(lens) + max_new - 1 > self.cfg.n_pos:
            raise ValueError(f"a prompt and its new tokens exceed the {self.cfg.n_pos} positions")
        if not 1 <= beams <= MAX_BEAMS or len(prompts) * beams > MAX_BATCH:
            raise ValueError(f"beams is 1 to {MAX_BEAMS}, and {MAX_BATCH} at most over all prompts")
        if not -1 <= eos < self.cfg.vocab:
            raise ValueError("eos is -1 or a token of the vocabulary")
        if chunk is not None and chunk < 1:
            raise ValueError("chunk is at least 1")
        cfg, B, W = self.cfg, len(prompts), beams
        table, owned, count = assign_pages(lens, W, max_new, self.page_size)
        table, owned = i32(table), i32(owned)
        shape = (cfg.n_layer, count, cfg.n_head, self.page_size, cfg.head_dim)
        kp = torch.empty(shape, dtype=self.cache_dtype, device=self.dev)
        vp = torch.empty_like(kp)
        logits = torch.empty((B * W, cfg.vocab), dtype=torch.float32, device=self.dev)

        # The prompts, through the first beams' tables. (A prompt that is done is left out of
        # the pass: the attention's kernel goes by the rows that a request has on average.)
        step = max(lens) if chunk is None else chunk
        for begin in range(0, max(lens), step):
            live = [b for b, n in enumerate(lens) if n > begin]
            parts = [np.asarray(prompts[b], np.int64)[begin:begin + step] for b in live]
            upto = list(itertools.accumulate(len(p) for p in parts))
            cu, kv_len, first = i32([0, *upto]), i32([begin + len(p) for p in parts]), table[i32(live).long() * W]
            ids = torch.from_numpy(np.concatenate(parts)).to(self.dev)
            at = torch.from_numpy(np.concatenate([np.arange(begin, begin + len(p)) for p in parts])).to(self.dev)
            attend = lambda i, q, k, v: serving.paged_attention(q, k, v, kp[i], vp[i], first, kv_len, cu,
                                                                workspace=self.attn_ws)
            x = self._pass(ids, at, attend)
            done = {b: upto[i] - 1 for i, b in enumerate(live) if lens[b] <= begin + step}  # last position, a row of x
            if done:
                rows = torch.tensor(list(done.values()), device=self.dev)
                logits[torch.tensor(list(done), device=self.dev) * W] = self._logits(x[rows])

        # The beams: only the first is in use, with a score of 0.
        scores = torch.full((B, W), float("-inf"), device=self.dev)
        scores[:, 0] = 0.0
        ended = torch.zeros((B, W), dtype=torch.uint8, device=self.dev)
        kv_len = i32(lens)
        rows_len, cu = kv_len.repeat_interleave(W), i32(np.arange(B * W + 1))
        parents = torch.zeros((max_new, B, W), dtype=torch.int32, device=self.dev)
        tokens = torch.zeros_like(parents)
        at = torch.zeros(1, dtype=torch.int64, device=self.dev)
        next_ids = torch.zeros(B * W, dtype=torch.int64, device=self.dev)

        def choose():
            s, parent, token, d = serving.beam_select(logits, scores, ended, eos, workspace=self.attn_ws)
            scores.copy_(s)
            ended.copy_(d)
            parents.index_copy_(0, at, parent[None])
            tokens.index_copy_(0, at, token[None])
            at.add_(1)
            next_ids.copy_(token.view(-1))
            if W > 1:
                serving.beam_reorder(parent, table, owned, kv_len, kp, vp)

        def decode():
            positions = rows_len.long()
            rows_len.add_(1)
            attend = lambda i, q, k, v: serving.paged_attention(q, k, v, kp[i], vp[i], table, rows_len, cu,
                                                                workspace=self.attn_ws)
            self._logits(self._pass(next_ids, positions, attend), out=logits)
            kv_len.add_(1)
            choose()

        choose()
        graph = None
        for i in range(max_new - 1):
            if graph is not None:
                graph.replay()
            elif use_graph and i == 1:  # the first step ran as it is and sized the workspaces
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    decode()
                graph.replay()
            else:
                decode()
        # Each beam's tokens, back through its parents.
        parents, tokens = parents.cpu().numpy(), tokens.cpu().numpy()
        out = np.zeros((B, W, max_new), np.int32)
        row = np.tile(np.arange(W), (B, 1))
        for i in reversed(range(max_new)):
            out[:, :, i] = np.take_along_axis(tokens[i], row, 1)
            row = np.take_along_axis(parents[i], row, 1)
        return {"tokens": out, "scores": scores.cpu().numpy()}
