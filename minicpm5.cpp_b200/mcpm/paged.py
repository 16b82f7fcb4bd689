"""Decoding over a bounded, paged KV cache, composed from the ops of include/mcpm.h.

`PagedDecoder` runs MiniCPM5 (Q4_K_M GGUF) for several sequences that share one pool of pages: each step
appends every sequence's K and V to its pages (`mcpm_paged_append`), attends over them while accumulating
attention mass (`mcpm_paged_attention`), and, where a sequence has outgrown its budget, moves its heaviest
positions to fresh pages (`mcpm_paged_evict`) and gives the old ones back.  Penalties, biases and grammar masks
are applied to the logits on the device (`mcpm_logits_process`) before the greedy token is taken.  Positions keep
counting past an eviction, so a conversation can outlive its cache (the reference stops at its context size,
src/ops/ops.cpp:550-553).

The projections are the single-vector GEMVs, one sequence after the other: for throughput over many sequences of
one length there is the engine's batched decode; this is the path for sequences of unlike and unbounded lengths.

    python -m mcpm.paged --tokens 64 --keep 48        # synthetic model, one sequence, greedy
"""
from __future__ import annotations

import argparse
import operator
import os
import time
from typing import Dict, List, Optional, Tuple

import numpy as np
import torch

from . import engine as E, gguf, spec, synth


def dequantize_q4_k(raw: np.ndarray) -> np.ndarray:
    """fp32 values of Q4_K super-blocks (reference include/ops.h:43-48), uint8 [n][144] -> float32 [n][256]."""
    d, dmin = (raw[:, i:i + 2].copy().view(np.float16).astype(np.float32) for i in (0, 2))
    q = raw[:, 4:16]   # eight 6-bit scales and mins
    scale = np.concatenate([q[:, :4] & 63, (q[:, 8:] & 15) | (q[:, :4] >> 6) << 4], 1).astype(np.float32)
    low = np.concatenate([q[:, 4:8] & 63, (q[:, 8:] >> 4) | (q[:, 4:8] >> 6) << 4], 1).astype(np.float32)
    nib = raw[:, 16:].reshape(-1, 4, 1, 32)   # 64 values a group: low nibbles, then high ones
    vals = np.concatenate([nib & 15, nib >> 4], 2).reshape(-1, 8, 32).astype(np.float32)
    return ((d * scale)[:, :, None] * vals - (dmin * low)[:, :, None]).reshape(-1, 256)


def model_tensors(path: str) -> Tuple[Dict[str, spec.TensorInfo], int]:
    """The tensors that a decoder reads, by name, and the number of layers.  Their shapes size every buffer of the
    kernels, so a file of another shape, or one that ends early, is refused here."""
    size = os.path.getsize(path)
    there = {t.name: t for t in gguf.read_header(path)[1]}
    n_layer = 0
    while f"blk.{n_layer}.attn_q.weight" in there:
        n_layer += 1
    emb = there.get("token_embd.weight")
    vocab = emb.dims[1] if emb is not None and len(emb.dims) == 2 else 0
    want = {"token_embd.weight": (spec.N_EMBD, vocab), "output.weight": (spec.N_EMBD, vocab), "output_norm.weight": (spec.N_EMBD,)}
    for i in range(n_layer):
        want.update({f"blk.{i}.{base}.weight": spec.layer_dims(base) for base in spec.LAYER_TENSORS})
    for name, dims in want.items():
        t = there.get(name)
        if not n_layer or not vocab or t is None or t.dims != dims:
            raise E.MCPMError(E.BAD_FILE, f"{name}: {'absent' if t is None else t.dims}, expected {dims}")
        types = (spec.GGML_F32,) if len(dims) == 1 else (spec.GGML_Q4_K,) if t is emb else (spec.GGML_Q4_K, spec.GGML_Q6_K)
        if t.ggml_type not in types:
            raise E.MCPMError(E.UNSUPPORTED_TYPE, f"{name}: the paged decoder reads Q4_K_M files")
        if t.offset + t.nbytes > size:
            raise E.MCPMError(E.BAD_FILE, f"{name}: beyond the end of the file")
    return {name: there[name] for name in want}, n_layer


class PagedDecoder:
    """keep: positions that a sequence has after an eviction, which comes when it reaches keep + slack of them
    (0: never evicted); sink and recent of them are always the first and the last ones.  rope_len: positions that the
    RoPE table has at first; it doubles when a sequence comes to its end (512 bytes a position).

    An eviction copies to ceil(keep / page_size) free pages before it frees the old ones, one sequence after the other:
    with max_seqs * ceil((keep + max(slack, 1)) / page_size) + ceil(keep / page_size) pages the pool never runs out.  A
    step that would need more than are free is refused as a whole (OOM)."""

    def __init__(self, path: str, n_pages: int, page_size: int = 16, max_seqs: int = 1, max_positions: int = 1024,
                 kv_type: int = E.KV_F32, keep: int = 0, slack: int = 16, sink: int = 4, recent: int = 16,
                 rope_len: int = 16384):
        max_pages = -(-max_positions // page_size)
        if keep and (min(keep, slack, sink, recent) < 0 or sink + recent > keep or keep + slack > max_positions or keep >= max_pages * page_size):
            raise ValueError("0 <= sink + recent <= keep, 0 <= slack, keep + slack <= max_positions, room for a position beyond keep")
        self.tensors, self.n_layer = model_tensors(path)
        emb = self.tensors["token_embd.weight"]
        self.n_vocab = emb.dims[1]
        self.file = np.memmap(path, np.uint8, "r")
        self.embeddings = self.file[emb.offset:emb.offset + emb.nbytes].reshape(self.n_vocab, -1, 144)
        # everything but the embeddings, as it lies in the file
        self.weights = {name: torch.from_numpy(np.array(self.file[t.offset:t.offset + t.nbytes])).cuda()
                        for name, t in self.tensors.items() if name != "token_embd.weight"}
        self.page_size, self.max_seqs, self.keep, self.slack, self.sink, self.recent = page_size, max_seqs, keep, slack, sink, recent
        self.max_positions = max_pages * page_size
        self.cfg = E.paged_config(kv_type, spec.N_HEAD, spec.N_HEAD_KV, spec.HEAD_DIM, page_size, n_pages, max_seqs, max_pages)
        dtype = {E.KV_F32: torch.float32, E.KV_F16: torch.float16, E.KV_BF16: torch.bfloat16}[kv_type]
        shape = (self.n_layer, n_pages, page_size, spec.N_HEAD_KV, spec.HEAD_DIM)
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2))
        self.mass = torch.zeros((self.n_layer, n_pages, spec.N_HEAD_KV, page_size), device="cuda")
        self.pools = [E.paged_pool(self.k[i].data_ptr(), self.v[i].data_ptr(), self.mass[i].data_ptr()) for i in range(self.n_layer)]
        self.workspace = torch.zeros(E.paged_workspace_bytes(self.cfg), dtype=torch.uint8, device="cuda")
        self.rope = self._rope_table(rope_len)
        # host state: a row per open sequence
        self.free: List[int] = list(range(n_pages))[::-1]
        self.table = np.full((max_seqs, max_pages), -1, np.int32)
        self.length = np.zeros(max_seqs, np.int32)     # positions in the cache
        self.position = np.zeros(max_seqs, np.int32)   # tokens seen, evicted ones among them
        self.opened: List[bool] = [False] * max_seqs
        self.history: List[List[int]] = [[] for _ in range(max_seqs)]
        f32 = dict(dtype=torch.float32, device="cuda")
        n = max_seqs
        self.x = torch.empty((n, spec.N_EMBD), **f32)
        self.qkv = torch.empty((n, spec.N_EMBD + 2 * spec.KV_DIM), **f32)
        self.q, self.att, self.y = (torch.empty((n, spec.N_EMBD), **f32) for _ in range(3))
        self.gate, self.up = (torch.empty(spec.N_FF, **f32) for _ in range(2))
        self.xq = torch.empty(spec.N_FF // 256 * 292, dtype=torch.uint8, device="cuda")
        self.logits, self.processed = (torch.empty((n, self.n_vocab), **f32) for _ in range(2))
        self.token = torch.empty(n, dtype=torch.int32, device="cuda")

    # ---------------------------------------------------------------- sequences and pages
    def open(self) -> int:
        for i, used in enumerate(self.opened):
            if not used:
                self.opened[i] = True
                self.length[i] = self.position[i] = 0
                self.history[i] = []
                return i
        raise E.MCPMError(E.BAD_ARG, "no free sequence")

    def _names_one(self, seq: int) -> bool:
        return 0 <= operator.index(seq) < self.max_seqs

    def close(self, seq: int) -> None:
        if not self._names_one(seq):
            raise E.MCPMError(E.BAD_ARG, f"sequence {seq}")
        self._give_back(seq)
        self.opened[seq] = False
        self.length[seq] = 0

    def _take(self, n: int) -> List[int]:
        if len(self.free) < n:
            raise E.MCPMError(E.OOM, "page pool exhausted")
        return [self.free.pop() for _ in range(n)]

    def _give_back(self, seq: int) -> None:
        self.free += [int(p) for p in self.table[seq] if p >= 0]
        self.table[seq] = -1

    def _dev(self, a: np.ndarray, dtype=np.int32) -> torch.Tensor:
        return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()

    def _evict(self, seq: int) -> None:
        """The sequence's self.keep heaviest positions of each layer and head, on fresh pages."""
        fresh = np.full((1, self.table.shape[1]), -1, np.int32)
        pages = self._take(-(-self.keep // self.page_size))
        fresh[0, :len(pages)] = pages
        src, dst, length = self._dev(self.table[seq:seq + 1]), self._dev(fresh), self._dev(self.length[seq:seq + 1])
        new_len = torch.empty(1, dtype=torch.int32, device="cuda")
        kept = torch.empty((1, spec.N_HEAD_KV, self.keep), dtype=torch.int32, device="cuda")
        for pool in self.pools:
            E.paged_evict(self.cfg, pool, src.data_ptr(), length.data_ptr(), dst.data_ptr(), new_len.data_ptr(), kept.data_ptr(), 1,
                          self.keep, self.sink, self.recent, self.workspace.data_ptr(), self.workspace.numel(), self._stream())
        self._give_back(seq)   # the copies are ordered before whatever is written to these pages next
        self.table[seq] = fresh[0]
        self.length[seq] = self.keep

    @staticmethod
    def _stream() -> int:
        return torch.cuda.current_stream().cuda_stream

    @staticmethod
    def _rope_table(n: int) -> torch.Tensor:
        return torch.from_numpy(E.rope_table(n, spec.HEAD_DIM, spec.ROPE_BASE)).cuda()

    def _reach(self, position: int) -> None:
        """Extends the RoPE table to a position: positions count on where the cache is bounded."""
        if position >= self.rope.shape[0]:
            self.rope = self._rope_table(max(2 * self.rope.shape[0], position + 1))

    # ---------------------------------------------------------------- one step
    def _needs_page(self, seq: int, length: int) -> bool:
        return length % self.page_size == 0 and self.table[seq, length // self.page_size] < 0

    def _check(self, tokens: Dict[int, int]) -> List[int]:
        """Raises where a step of these tokens cannot be made, before anything has changed; else the sequences that it
        evicts.  Pages are counted in the step's own order: an eviction takes its fresh ones before it frees the old."""
        evicted, free = [], len(self.free)
        for s, token in tokens.items():
            if not self._names_one(s) or not self.opened[s]:
                raise E.MCPMError(E.BAD_ARG, f"sequence {s}")
            if not 0 <= operator.index(token) < self.n_vocab:
                raise E.MCPMError(E.BAD_TOKEN, f"sequence {s}")
            length, fresh = int(self.length[s]), 0
            if self.keep and length >= self.keep + self.slack:
                evicted.append(s)
                fresh, length = -(-self.keep // self.page_size), self.keep
            if length >= self.max_positions:
                raise E.MCPMError(E.CTX_OVERFLOW, f"sequence {s}")
            more = length % self.page_size == 0 if fresh else self._needs_page(s, length)
            held = int((self.table[s] >= 0).sum()) if fresh else 0
            if free < fresh or free - fresh + held < more:
                raise E.MCPMError(E.OOM, f"page pool exhausted, sequence {s}")
            free += held - fresh - more
        return evicted

    def _admit(self, seqs: List[int], evicted: List[int]) -> None:
        """Makes room for one more position of each sequence, as _check has found possible."""
        for s in seqs:
            if s in evicted:
                self._evict(s)
            if self._needs_page(s, self.length[s]):
                self.table[s, self.length[s] // self.page_size] = self._take(1)[0]

    def _options(self, tokens: Dict[int, int], repetition: float, frequency: float, presence: float,
                 bias: Optional[Dict[int, float]], allow: Optional[np.ndarray]) -> Tuple[List[torch.Tensor], Dict[str, int]]:
        """The lists and masks of a step's logits on the device, and the arguments that name them.  Raises where they
        cannot be made, so that what is wrong with them is found before the step begins."""
        n, held, more = len(tokens), [], {}
        if (repetition, frequency, presence) != (1.0, 0.0, 0.0):
            if not repetition > 0:
                raise E.MCPMError(E.BAD_ARG, "repetition > 0")
            rows = [self.history[s][1 - E.MAX_HIST:] + [t] for s, t in tokens.items()]
            hist = np.full((n, max(map(len, rows))), -1, np.int32)
            for r, row in enumerate(rows):
                hist[r, :len(row)] = row
            held += [self._dev(hist), self._dev(np.tile(np.array([repetition, frequency, presence]), (n, 1)), np.float32)]
            more.update(hist=held[0].data_ptr(), hist_stride=hist.shape[1], penalties=held[1].data_ptr())
        if bias:
            if len(bias) > E.MAX_BIAS:
                raise E.MCPMError(E.BAD_ARG, f"more than {E.MAX_BIAS} biases")
            ids = np.array([t if 0 <= t < self.n_vocab else -1 for t in bias])   # foreign ids are ignored
            held += [self._dev(np.tile(ids, (n, 1))), self._dev(np.tile(np.array(list(bias.values())), (n, 1)), np.float32)]
            more.update(bias_token=held[-2].data_ptr(), bias=held[-1].data_ptr(), bias_stride=len(bias))
        if allow is not None:
            words = np.zeros((n, (self.n_vocab + 31) // 32 * 32), bool)
            words[:, :self.n_vocab] = allow
            held.append(self._dev(np.packbits(words, axis=1, bitorder="little").view(np.int32)))
            more.update(allow=held[-1].data_ptr())
        return held, more

    def _gemv(self, name: str, xq: torch.Tensor, out_ptr: int) -> None:
        t = self.tensors[name]
        E.gemv_q8k_block(t.ggml_type, self.weights[name].data_ptr(), xq.data_ptr(), out_ptr, t.dims[1], t.dims[0], self._stream())

    def step(self, tokens: Dict[int, int], repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0,
             bias: Optional[Dict[int, float]] = None, allow: Optional[np.ndarray] = None) -> Dict[int, int]:
        """Feeds one token to each given sequence and returns their greedy next tokens (-1: the grammar allows none).
        Penalties count the tokens fed so far (the last 1048575 of them; the lists are laid out and copied anew in each
        step that has penalties); allow: bool [n_vocab] or [len(tokens)][n_vocab]."""
        seqs = list(tokens)
        n = len(seqs)
        evicted = self._check(tokens)
        held, more = self._options(tokens, repetition, frequency, presence, bias, allow)   # held: the lists' memory
        self._reach(max(int(self.position[s]) for s in seqs))
        self._admit(seqs, evicted)
        st, ws = self._stream(), (self.workspace.data_ptr(), self.workspace.numel())
        table, slot = self._dev(self.table[seqs]), self._dev(self.length[seqs])
        pos, length = self._dev(self.position[seqs]), self._dev(self.length[seqs] + 1)
        rows = dequantize_q4_k(np.concatenate([self.embeddings[tokens[s]] for s in seqs]))
        x = self.x[:n].copy_(torch.from_numpy(rows.reshape(n, spec.N_EMBD)))
        w, xq, wide = self.weights, self.xq, 4 * self.qkv.shape[1]
        for i in range(self.n_layer):
            b = f"blk.{i}."
            for r in range(n):
                E.rmsnorm_q8k(x[r].data_ptr(), w[b + "attn_norm.weight"].data_ptr(), xq.data_ptr(), spec.N_EMBD, spec.RMS_EPS, st)
                out = self.qkv.data_ptr() + r * wide
                for name, at in (("attn_q", 0), ("attn_k", spec.N_EMBD), ("attn_v", spec.N_EMBD + spec.KV_DIM)):
                    self._gemv(b + name + ".weight", xq, out + 4 * at)
            q = self.qkv.data_ptr()
            E.paged_append(self.cfg, self.pools[i], table.data_ptr(), n, slot.data_ptr(), q + 4 * spec.N_EMBD,
                           q + 4 * (spec.N_EMBD + spec.KV_DIM), tok_pos=pos.data_ptr(), q=q, q_out=self.q.data_ptr(), q_stride=wide // 4,
                           kv_stride=wide // 4, rope=self.rope.data_ptr(), rope_len=self.rope.shape[0], n_seq=n, stream=st)
            E.paged_attention(self.cfg, self.pools[i], table.data_ptr(), length.data_ptr(), n, self.q.data_ptr(), self.att.data_ptr(), *ws, stream=st)
            for r in range(n):
                E.quantize_q8k(self.att[r].data_ptr(), xq.data_ptr(), spec.N_EMBD, E.ROUND_EVEN, st)
                self._gemv(b + "attn_output.weight", xq, self.y[r].data_ptr())
            x += self.y[:n]
            for r in range(n):
                E.rmsnorm_q8k(x[r].data_ptr(), w[b + "ffn_norm.weight"].data_ptr(), xq.data_ptr(), spec.N_EMBD, spec.RMS_EPS, st)
                self._gemv(b + "ffn_gate.weight", xq, self.gate.data_ptr())
                self._gemv(b + "ffn_up.weight", xq, self.up.data_ptr())
                E.swiglu_q8k(self.gate.data_ptr(), self.up.data_ptr(), xq.data_ptr(), spec.N_FF, st)
                self._gemv(b + "ffn_down.weight", xq, self.y[r].data_ptr())
            x += self.y[:n]
        for r, s in enumerate(seqs):
            E.rmsnorm_q8k(x[r].data_ptr(), w["output_norm.weight"].data_ptr(), xq.data_ptr(), spec.N_EMBD, spec.RMS_EPS, st)
            self._gemv("output.weight", xq, self.logits[r].data_ptr())
            self.length[s] += 1
            self.position[s] += 1
            self.history[s].append(tokens[s])
        E.logits_process(self.logits.data_ptr(), self.processed.data_ptr(), n, self.n_vocab, argmax=self.token.data_ptr(), stream=st, **more)
        return dict(zip(seqs, self.token[:n].tolist()))


def main() -> None:
    ap = argparse.ArgumentParser(description="greedy decoding of the synthetic model over a bounded paged cache")
    ap.add_argument("--model", default=None, help="Q4_K_M GGUF file (default: the synthetic one)")
    ap.add_argument("--prompt", type=int, default=16, help="prompt tokens")
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--keep", type=int, default=48, help="positions after an eviction; 0: unbounded")
    ap.add_argument("--repetition", type=float, default=1.1)
    a = ap.parse_args()
    path = a.model or synth.ensure_model("q4_k_m", 0, dscale=0.04)   # logits that depend on the input
    total = a.prompt + a.tokens
    d = PagedDecoder(path, n_pages=total // 16 + 16, max_positions=max(total, a.keep + 16), keep=a.keep, recent=min(16, a.keep // 2), sink=min(4, a.keep // 4))
    s = d.open()
    token = -1
    for t in synth.prompt_ids(a.prompt):
        token = d.step({s: int(t)}, repetition=a.repetition)[s]
    out = []
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.tokens):
        out.append(token)
        token = d.step({s: token}, repetition=a.repetition)[s]
    torch.cuda.synchronize()
    ms = (time.perf_counter() - began) / max(1, a.tokens) * 1e3
    print(f"{total} tokens, {d.length[s]} positions in {int((d.table[s] >= 0).sum())} pages, {ms:.2f} ms per token")
    print(*out)


if __name__ == "__main__":
    main()
